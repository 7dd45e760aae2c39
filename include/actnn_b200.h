/*
 * actnn_b200 -- C ABI of the B200 (sm_100a) activation compress / decompress kernels.
 *
 * Drop-in boundary for the native extensions of ucbrise/actnn
 * (actnn/actnn/cpp_extension/{minimax,quantization,calc_precision}*).  The reference
 * binds those as pybind11 torch extensions that take and return torch::Tensor; this
 * library exposes the same operations one level lower: plain device pointers, explicit
 * sizes, a dtype tag and a cudaStream_t.  A binding layer (python/ctypes here, or the
 * reference's own .cc files) allocates the outputs and forwards the pointers.
 *
 * Conventions
 *   - every pointer is a device pointer on the current device unless stated otherwise;
 *   - no entry point allocates, frees or synchronises; all work is queued on `stream`;
 *   - every entry point returns an actnn_status (0 = queued successfully); arguments are
 *     validated on the host before anything is launched;
 *   - activations are viewed as [N, G, group_size] (sample, group, element), contiguous,
 *     each sample zero-padded to a whole number of groups by the caller, as the
 *     reference's schemes do (actnn/actnn/qscheme.py:61-71);
 *   - `dtype` is the element type of the activation; per-group statistics (min, max,
 *     scale) carry `stat_dtype`, which equals `dtype` except that float32 activations may
 *     keep bfloat16 statistics (the reference's storage format, actnn/actnn/ops.py:115-116);
 *   - the arithmetic is the reference's "simulate" branch (actnn/actnn/ops.py:23-41,56-57)
 *     with every intermediate rounded to `dtype`, so codes and packed bytes are bit-exact
 *     against it for the same rounding noise;
 *   - rounding noise: pass `noise` (device array, same shape and dtype as the activation,
 *     values in [-0.5, 0.5]) to inject it, or NULL to draw it in registers from
 *     Philox4x32-10 keyed by (seed, offset); actnn_noise_fill() materialises exactly that
 *     stream.  `stochastic == 0` rounds to nearest without noise.
 *   - a NaN input yields some valid code (0 or the largest); it never corrupts its neighbours.
 */
#ifndef ACTNN_B200_H_
#define ACTNN_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* actnn_stream_t;        /* == cudaStream_t */

typedef enum {
  ACTNN_F32 = 0,
  ACTNN_F16 = 1,
  ACTNN_BF16 = 2
} actnn_dtype;

typedef enum {
  ACTNN_OK = 0,
  ACTNN_ERR_NULL = 1,         /* a required pointer is NULL */
  ACTNN_ERR_DTYPE = 2,        /* dtype / stat_dtype not supported by this entry point */
  ACTNN_ERR_SHAPE = 3,        /* negative size, size overflow, unsupported group size */
  ACTNN_ERR_BITS = 4,         /* bit width outside the supported set */
  ACTNN_ERR_ALIGN = 5,        /* pointer not aligned for vector access */
  ACTNN_ERR_ARG = 6,          /* any other invalid argument (e.g. stochastic rounding off where the reference requires it) */
  ACTNN_ERR_LAUNCH = 7,       /* the CUDA runtime refused the launch; see cudaGetLastError() */
  ACTNN_ERR_CAPACITY = 8      /* problem larger than a fixed internal buffer */
} actnn_status;

/* Human-readable text for a status code (static storage). */
const char* actnn_status_string(int status);
/* Library ABI version, bumped on any signature change. */
int actnn_abi_version(void);

/* ------------------------------------------------------------------------------------
 * Per-group min / max.
 * Replaces: minimax(data) -> (min, max), actnn/actnn/cpp_extension/minimax.cc:7-11 and
 * minimax_cuda_kernel.cu:23-89.  data[rows, cols] -> mn[rows], mx[rows], all `dtype`.
 * The reference requires cols % 32 == 0 && cols > 32; so does this.  cols == 256 takes
 * the vectorised path (one warp per row, 128/256-bit loads).
 */
int actnn_minimax(const void* data, void* mn, void* mx, int64_t rows, int64_t cols,
                  int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Mixed-precision bit stream (per-sample bit widths, int32 words).
 * Layout (actnn/actnn/cpp_extension/quantization_cuda_kernel.cu:51-79): the block of
 * (sample n, group g) starts at word (P[n-1]*G*gs + bits[n]*g*gs) / 32, P the inclusive
 * prefix sum of bits; bit i of element d sits in word (d*b+i) % W at bit (d*b+i) / W,
 * W = gs*b/32.
 *
 * actnn_bits_prefix: word_offsets[n] = first word of sample n, word_offsets[N] = total
 * words.  Replaces the torch::cumsum + .item() of quantization_cuda_kernel.cu:97-98 /
 * :182 without a host sync.  One thread block; N <= 2^20.
 */
int actnn_bits_prefix(const int32_t* bits, int64_t N, int64_t G, int64_t group_size,
                      int64_t* word_offsets, actnn_stream_t stream);

/* Replaces: pack_mixed_precision(data, min, max, bits, stochastic) -> (packed, scale),
 * actnn/actnn/cpp_extension/quantization.cc:46-57, quantization_cuda_kernel.cu:37-142.
 * data[N,G,gs], mn/mx[N,G] in `dtype`; bits[N] in 1..8; word_offsets from
 * actnn_bits_prefix; writes packed (word_offsets[N] words) and scale[N,G] (`stat_dtype`).
 * If mn_out is not NULL the minimum is also re-written there in `stat_dtype`.
 * group_size must be 256. */
int actnn_pack_mixed(const void* data, const void* mn, const void* mx, const int32_t* bits,
                     const int64_t* word_offsets, int32_t* packed, void* scale, void* mn_out,
                     int64_t N, int64_t G, int64_t group_size, int dtype, int stat_dtype,
                     int stochastic, const void* noise, uint64_t seed, uint64_t offset,
                     actnn_stream_t stream);

/* Replaces: unpack_mixed_precision(data, bits, scale, min, N, num_groups, group_size),
 * actnn/actnn/cpp_extension/quantization.cc:59-73, quantization_cuda_kernel.cu:145-205.
 * out[N,G,gs] in `dtype` = code / scale + min. */
int actnn_unpack_mixed(const int32_t* packed, const int32_t* bits, const int64_t* word_offsets,
                       const void* scale, const void* mn, void* out,
                       int64_t N, int64_t G, int64_t group_size, int dtype, int stat_dtype,
                       actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Single-precision (uniform bit width) byte stream, int8.
 * Layout (quantization_cuda_kernel.cu:236-257): byte (no*G + g)*gs + d holds samples
 * no*wpt + ni (wpt = 8 / bits) at bit offset ni*bits; length
 * bits * N_round * G * gs / 8 + 1 with N rounded up to a multiple of wpt (the trailing
 * byte is written as zero).  bits in {1, 2, 4, 8}; group_size must be 256.
 *
 * Replaces: pack_single_precision(data, min, max, bits, stochastic) -> (packed, scale),
 * actnn/actnn/cpp_extension/quantization.cc:77-87, quantization_cuda_kernel.cu:225-330. */
int actnn_pack_single(const void* data, const void* mn, const void* mx, int bits,
                      int8_t* packed, void* scale, void* mn_out,
                      int64_t N, int64_t G, int64_t group_size, int dtype, int stat_dtype,
                      int stochastic, const void* noise, uint64_t seed, uint64_t offset,
                      actnn_stream_t stream);

/* Replaces: unpack_single_precision(data, bits, scale, min, N, num_groups, group_size),
 * actnn/actnn/cpp_extension/quantization.cc:89-102, quantization_cuda_kernel.cu:333-405. */
int actnn_unpack_single(const int8_t* packed, int bits, const void* scale, const void* mn,
                        void* out, int64_t N, int64_t G, int64_t group_size, int dtype,
                        int stat_dtype, actnn_stream_t stream);

/* Fused single pass: per-group min/max + stochastic rounding + pack, reading the
 * activation once.  Replaces the sequence minimax -> pack_single_precision that
 * no_scheme_compute_quantization_bits + quantize_and_pack issue for uniform-bit layers
 * (actnn/actnn/ops.py:77-96, 44-48).  Writes packed, scale[N,G] and mn[N,G]
 * (`stat_dtype`); mx_out may be NULL. */
int actnn_compress_single(const void* data, int bits, int8_t* packed, void* scale, void* mn_out,
                          void* mx_out, int64_t N, int64_t G, int64_t group_size, int dtype,
                          int stat_dtype, int stochastic, const void* noise, uint64_t seed,
                          uint64_t offset, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Bit allocation on the device.
 *
 * actnn_range_sqr: per-sample sensitivity base, Range_sqr[n] =
 * float(norm_T(mx[n,:] - mn[n,:]))^2 * (group_size / num_pixels), the expression of
 * actnn/actnn/qscheme.py:80 / qbnscheme.py:42; then C[n] = coeff * Range_sqr[n] *
 * (grad_scale ? *grad_scale : 1) in float32 (qscheme.py:84).  grad_scale is a device
 * pointer to one float or NULL. */
int actnn_range_sqr(const void* mn, const void* mx, int64_t N, int64_t G, int stat_dtype,
                    float range_factor, float coeff, const float* grad_scale, float* C,
                    actnn_stream_t stream);

/* Per-sample squared gradient norm, out[n] = sum_f float(grad[n, f])^2.
 * Replaces the torch expression of QScheme.set_scale, actnn/actnn/qscheme.py:47-55
 * (grad.view(N, -1).float().norm(dim=1).square()) with one read of the gradient. */
int actnn_sample_sumsq(const void* grad, float* out, int64_t N, int64_t F, int dtype,
                       actnn_stream_t stream);
/* The same and *mean, the mean of out[0..N-1] (qscheme.py:55), N >= 1.  `ticket`: as in
 * actnn_compress_mixed_prestat_kept. */
int actnn_sample_sumsq_mean(const void* grad, float* out, float* mean, void* ticket, int64_t N, int64_t F, int dtype,
                            actnn_stream_t stream);

/* Replaces: calc_precision(b, C, w, target) -> b,
 * actnn/actnn/cpp_extension/calc_precision.cc:9-50 (a CPU priority queue there; here a
 * weighted radix select over the (initial_bits-1)*N candidate decrements, identical
 * results including tie-breaks).  C[N] float32, w[N] int32 or NULL (all ones),
 * b_out[N] int32, every entry starting from `initial_bits` (1..15; 1 leaves nothing to remove).  If word_offsets is
 * not NULL it receives what actnn_bits_prefix would (needs G, group_size).
 * N <= 2^20.  Small unit-weight problems run in one thread block.  `workspace` (optional,
 * actnn_calc_precision_workspace() bytes, 8-byte aligned, contents unspecified before and
 * after) lets weighted or large problems without word offsets run as a sequence of
 * multi-block launches instead of one block; pass NULL / 0 to do without. */
int64_t actnn_calc_precision_workspace(void);
int actnn_calc_precision(const float* C, const int32_t* w, int64_t N, int initial_bits,
                         double target, int32_t* b_out, int64_t* word_offsets,
                         int64_t G, int64_t group_size, void* workspace, int64_t workspace_bytes,
                         actnn_stream_t stream);

/* The joint allocation over layers x samples that a step ends with (QScheme.allocate_perlayer,
 * actnn/actnn/qscheme.py:96-128): actnn_calc_precision over the concatenation of L sensitivity vectors C[l][N] with
 * the weight dims[l] > 0 for layer l's samples, and the sum of the widths of each layer's samples, sums[L].  C and dims
 * are host arrays (of device pointers / values), read before the call returns.  One launch.  initial_bits 1..8;
 * ACTNN_ERR_CAPACITY for L > 256 or N * L > 32768 (take actnn_calc_precision then). */
int actnn_allocate_layers(const float* const* C, const int32_t* dims, int L, int64_t N, int initial_bits,
                          double target, int32_t* sums, actnn_stream_t stream);

/* The adaptive compress of one activation as one call: per-group min/max, sensitivities,
 * greedy allocation at `target` total bits, scale + stochastic rounding + mixed-precision
 * pack.  Replaces the sequence QScheme.compute_quantization_bits -> quantize_and_pack,
 * actnn/actnn/qscheme.py:57-94 and actnn/actnn/ops.py:44-48 (there: ~15 launches, two host
 * copies and a CPU heap).  Outputs: packed (the caller sizes it for the bit total the greedy
 * will reach: min(initial_bits*N, max(target, N)) * G * group_size / 32 words), scale and
 * mn_out [N,G] (`stat_dtype`), bits_out [N], word_offsets_out [N+1], C_out [N] (float32
 * sensitivities, kept by the caller for the per-layer allocation).
 * `workspace` is caller-provided scratch of at least actnn_compress_mixed_workspace(N, G,
 * dtype) bytes, 256-byte aligned; it holds the per-group min / max between the kernels and
 * its content afterwards is unspecified.  Arguments otherwise as in actnn_range_sqr,
 * actnn_calc_precision and actnn_pack_mixed. */
int64_t actnn_compress_mixed_workspace(int64_t N, int64_t G, int dtype);
int actnn_compress_mixed(const void* data, int32_t* packed, void* scale, void* mn_out,
                         int32_t* bits_out, int64_t* word_offsets_out, float* C_out,
                         void* workspace, int64_t workspace_bytes, int64_t N, int64_t G,
                         int64_t group_size, int dtype, int stat_dtype, float range_factor,
                         float coeff, const float* grad_scale, int initial_bits, double target,
                         int stochastic, const void* noise, uint64_t seed, uint64_t offset,
                         actnn_stream_t stream);

/* actnn_compress_mixed and actnn_unpack_mixed on samples of any length: data / out are [N, F], contiguous,
 * groups are 256 elements, G = ceil(F / 256), and the last group of a sample is completed with zeros, as the
 * reference's padding does (actnn/actnn/qscheme.py:61-71, stripped again in ops.py:137-139), without a padded copy.
 * data / out need the alignment of one element only.  `noise`, when given, is [N, G, 256]. */
int actnn_compress_mixed_samples(const void* data, int32_t* packed, void* scale, void* mn_out,
                                 int32_t* bits_out, int64_t* word_offsets_out, float* C_out,
                                 void* workspace, int64_t workspace_bytes, int64_t N, int64_t F, int dtype,
                                 int stat_dtype, float range_factor, float coeff, const float* grad_scale,
                                 int initial_bits, double target, int stochastic, const void* noise,
                                 uint64_t seed, uint64_t offset, actnn_stream_t stream);
int actnn_unpack_mixed_samples(const int32_t* packed, const int32_t* bits, const int64_t* word_offsets,
                               const void* scale, const void* mn, void* out, int64_t N, int64_t F, int dtype,
                               int stat_dtype, actnn_stream_t stream);

/* actnn_compress_mixed for callers that cannot hand over scratch memory.  (This entry point
 * has no counterpart in the reference.)
 * Who needs it: code that only works with pointers it was given -- a plug-in of a host
 * framework that owns all device memory and offers no allocator, or a job whose device
 * memory was planned out in advance so that one more cudaMalloc may fail or upset the plan.
 * Same arguments and results as actnn_compress_mixed without `workspace`: the per-group
 * min / max go to an array of actnn_compress_mixed_static_capacity() bytes (4 MiB + 256) that is
 * part of the library image, i.e. resident on every GPU that loads the library until the
 * process ends.  Limits and rules:
 *   - actnn_compress_mixed_workspace(N, G, dtype) must not exceed the capacity (N*G up to
 *     1 Mi groups of 16-bit data, 512 Ki of float32); larger problems return
 *     ACTNN_ERR_CAPACITY and nothing is launched;
 *   - the first call on a device looks up the array's device address (with that device
 *     current); make that first call before any stream capture begins;
 *   - every call on a device uses the same array and leaves its last contents behind (no
 *     part of it needs clearing: each call overwrites what it reads); two calls that may
 *     overlap on the GPU (different streams) race on it -- serialise them;
 *   - it never calls cudaMalloc, cudaFree or any allocating routine. */
int64_t actnn_compress_mixed_static_capacity(void);
int actnn_compress_mixed_static(const void* data, int32_t* packed, void* scale, void* mn_out,
                                int32_t* bits_out, int64_t* word_offsets_out, float* C_out,
                                int64_t N, int64_t G, int64_t group_size, int dtype, int stat_dtype,
                                float range_factor, float coeff, const float* grad_scale,
                                int initial_bits, double target, int stochastic, const void* noise,
                                uint64_t seed, uint64_t offset, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Batch-norm statistics and the codec's per-group min / max from ONE read of x.
 * Replaces, for a quantized batch norm in training mode, the pair of reads the reference
 * makes: the statistics inside at::cudnn_batch_norm (backward_func.cc:87, called at
 * actnn/actnn/ops.py:456-458; torch.batch_norm_stats at ops.py:515 for the synchronised
 * layer) and the min / max of QBNScheme.compute_quantization_bits (qbnscheme.py:28-40).
 *   x           [N, C, HW] contiguous (NCHW), dtype float32 / float16 / bfloat16
 *   mn, mx      [N * C * HW / 256] in x's dtype: min / max of every 256-element group of the
 *               flattened samples (what actnn_minimax returns for the same tensor)
 *   save_mean, save_invstd  float32 [C]; running_mean / running_var (may be NULL) are updated
 *               with `momentum` exactly as actnn_batch_norm_forward does
 *   weight, bias  not read; may be NULL
 * Geometry: HW % 8 == 0, HW >= 256 and C * HW % 256 == 0 (every layer of a ResNet down to
 * 16x16 maps); anything else returns ACTNN_ERR_SHAPE and the caller takes the two-read path.
 * actnn_batch_norm_stats_minimax_workspace returns the scratch bytes (-1: unsupported). */
int64_t actnn_batch_norm_stats_minimax_workspace(int64_t N, int64_t C, int64_t HW);
int actnn_batch_norm_stats_minimax(const void* x, void* mn, void* mx, const float* weight, const float* bias,
                                   float* running_mean, float* running_var, float* save_mean, float* save_invstd,
                                   int64_t N, int64_t C, int64_t HW, double momentum, double eps, int dtype,
                                   void* workspace, int64_t workspace_bytes, actnn_stream_t stream);

/* [batch, rows, cols] -> [batch, cols, rows] for 16-bit elements: NCHW <-> NHWC around the convolution
 * library (reference call sites: actnn/actnn/ops.py:163-220).  in and out must not overlap. */
int actnn_transpose16(const void* in, void* out, int64_t batch, int64_t rows, int64_t cols, actnn_stream_t stream);

/* The backward half of a training-mode batch norm straight from the compressed activation (mixed stream, groups of 256
 * over samples of C * HW elements, as actnn_compress_mixed / actnn_compress_mixed_samples write them).  Replaces
 * unpack + batch-norm backward, actnn/actnn/ops.py:470-493: the decoded activation only exists in registers.
 * Arguments as in actnn_unpack_mixed and actnn_batch_norm_backward; stat_dtype is `dtype`, or bfloat16 for float32.
 * Any C, HW >= 8.  grad_out / grad_in need the alignment of one element.  Scratch: *bytes of the first call (a host
 * pointer; ACTNN_ERR_SHAPE: not covered), 16-byte aligned, for the current device. */
int actnn_batch_norm_codes_workspace(int64_t N, int64_t C, int64_t HW, int dtype, int64_t* bytes);
/* The forward half: statistics, widths, codes and y = normalised x from two reads of x.  Replaces the compress of the
 * input followed by the batch norm, actnn/actnn/ops.py:446-458 and qbnscheme.py:28-52.  Outputs as in
 * actnn_compress_mixed_samples (coeff 1, no grad_scale, no injected noise) and actnn_batch_norm_forward; same
 * geometry and scratch as the backward half, the scratch 256-byte aligned.  With group_mn / group_mx (what
 * actnn_batch_norm_stats_minimax wrote; else both NULL) save_mean and save_invstd are inputs, too, and the running
 * statistics are left alone.  `ticket`: as in actnn_compress_mixed_prestat_kept. */
int actnn_batch_norm_codes_forward(const void* x, const void* group_mn, const void* group_mx, const float* weight,
                                   const float* bias, float* running_mean, float* running_var, void* y,
                                   float* save_mean, float* save_invstd, int32_t* packed,
                                   void* scale, void* mn_out, int32_t* bits_out, int64_t* word_offsets_out,
                                   float* C_out, int64_t N, int64_t C, int64_t HW, double momentum, double eps,
                                   int dtype, int stat_dtype, float range_factor, int initial_bits, double target,
                                   int stochastic, uint64_t seed, uint64_t offset, void* ticket, void* workspace,
                                   int64_t workspace_bytes, actnn_stream_t stream);
int actnn_batch_norm_codes_backward(const int32_t* packed, const int32_t* bits, const int64_t* word_offsets,
                                    const void* scale, const void* mn, const void* grad_out, const float* weight,
                                    const float* save_mean, const float* save_invstd, void* grad_in,
                                    float* grad_weight, float* grad_bias, int64_t N, int64_t C, int64_t HW, int dtype,
                                    int stat_dtype, void* workspace, int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * actnn_compress_mixed for an activation whose per-group min / max are already known (from
 * actnn_batch_norm_stats_minimax or actnn_minimax): sensitivities, greedy allocation and pack,
 * i.e. QBNScheme.compute_quantization_bits from its line qbnscheme.py:42 on, followed by
 * pack_mixed_precision (quantization.cc:46-57).  `mn` / `mx` must be the true group extrema.
 * `ticket_workspace`: 256 bytes of scratch, 256-byte aligned.  Other arguments as
 * actnn_compress_mixed. */
int actnn_compress_mixed_prestat(const void* data, const void* mn, const void* mx, int32_t* packed, void* scale,
                                 void* mn_out, int32_t* bits_out, int64_t* word_offsets_out, float* C_out,
                                 void* ticket_workspace, int64_t N, int64_t G, int64_t group_size, int dtype,
                                 int stat_dtype, float range_factor, float coeff, const float* grad_scale,
                                 int initial_bits, double target, int stochastic, const void* noise, uint64_t seed,
                                 uint64_t offset, actnn_stream_t stream);

/* actnn_compress_mixed_prestat (same replaced reference code: qbnscheme.py:42-52, quantization.cc:46-57) with a
 * ticket word that the caller keeps for this purpose only: zero before the first call, left at zero by every
 * call, touched by nothing else, used by one stream at a time.  The per-call clear of the ticket is skipped. */
int actnn_compress_mixed_prestat_kept(const void* data, const void* mn, const void* mx, int32_t* packed, void* scale,
                                      void* mn_out, int32_t* bits_out, int64_t* word_offsets_out, float* C_out,
                                      void* ticket_workspace, int64_t N, int64_t G, int64_t group_size, int dtype,
                                      int stat_dtype, float range_factor, float coeff, const float* grad_scale,
                                      int initial_bits, double target, int stochastic, const void* noise,
                                      uint64_t seed, uint64_t offset, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Mask ops.  The saved mask is 1 bit per element: bit (e % 8) of byte e / 8, padded to
 * whole int32 words (mask_words = ceil(numel / 32)).
 *
 * Replaces: act_quantized_relu forward / backward,
 * actnn/actnn/cpp_extension/quantization.cc:106-124, quantization_cuda_kernel.cu:411-508. */
int actnn_relu_forward(const void* x, void* y, int32_t* mask, int64_t numel, int dtype,
                       actnn_stream_t stream);

/* The same pass, which also leaves the min and the max of every 256 consecutive OUTPUTS in mn[g] / mx[g]
 * (g = element / 256; numel % 256 == 0), bit-identical to actnn_minimax(y).  The layer that consumes y
 * (a convolution: actnn/actnn/ops.py:99-118 quantizes its input with QScheme.compute_quantization_bits,
 * qscheme.py:57-94, whose first step is that min / max pass) can then compress it with
 * actnn_compress_mixed_prestat, i.e. without reading y once more for the ranges. */
int actnn_relu_forward_minimax(const void* x, void* y, int32_t* mask, void* mn, void* mx, int64_t numel,
                               int dtype, actnn_stream_t stream);
int actnn_relu_backward(const void* grad_out, const int32_t* mask, void* grad_in,
                        int64_t numel, int dtype, actnn_stream_t stream);

/* Replaces: act_quantized_dropout forward / backward,
 * actnn/actnn/cpp_extension/quantization.cc:128-148, quantization_cuda_kernel.cu:514-627.
 * keep = u > p with u uniform in (0, 1] from Philox (seed, offset), or from the injected
 * float32 array `u`; y = keep ? x / (1 - p) : 0. */
int actnn_dropout_forward(const void* x, void* y, int32_t* mask, int64_t numel, float p,
                          int dtype, const float* u, uint64_t seed, uint64_t offset,
                          actnn_stream_t stream);
int actnn_dropout_backward(const void* grad_out, const int32_t* mask, void* grad_in,
                           int64_t numel, float p, int dtype, actnn_stream_t stream);
/* The uniforms actnn_dropout_forward draws for (seed, offset), as float32. */
int actnn_dropout_uniform_fill(float* u, int64_t numel, uint64_t seed, uint64_t offset,
                               actnn_stream_t stream);

/* Replaces: act_quantized_max_pool2d forward / backward,
 * actnn/actnn/cpp_extension/quantization.cc:152-196, quantization_cuda_kernel.cu:633-754.
 * NCHW; saves the window-local arg-max kh*KW + kw as int8 per output; KH*KW < 16 as in
 * the reference.  Backward gathers (each input sums the windows that selected it), so
 * grad_in needs no zero fill and the result is deterministic. */
int actnn_max_pool2d_forward(const void* x, void* y, int8_t* idx, int64_t N, int64_t C,
                             int64_t H, int64_t W, int KH, int KW, int SH, int SW, int PH,
                             int PW, int DH, int DW, int dtype, actnn_stream_t stream);
int actnn_max_pool2d_backward(const void* grad_out, const int8_t* idx, void* grad_in,
                              int64_t N, int64_t C, int64_t H, int64_t W, int KH, int KW,
                              int SH, int SW, int PH, int PW, int DH, int DW, int dtype,
                              actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Training-mode batch normalisation of an NCHW tensor viewed as [N, C, HW] (HW = 1 for a
 * [N, C] input).  Replaces the cuDNN calls the reference's quantized batch-norm operator
 * makes: ext_backward_func.cudnn_batch_norm / cudnn_batch_norm_backward, re-exported at
 * actnn/actnn/cpp_extension/backward_func.cc:87-88 and called at actnn/actnn/ops.py:457-458
 * and actnn/actnn/ops.py:492-493.  Same results (batch statistics with the biased variance,
 * running statistics updated with `momentum` and the unbiased variance, save_mean and
 * save_invstd = 1/sqrt(var + eps) for backward); statistics, weight, bias and their
 * gradients are float32 whatever `dtype` is.  weight / bias NULL mean 1 / 0;
 * running_mean / running_var NULL skip the update; grad_in / grad_weight / grad_bias NULL
 * skip that output.  `workspace` holds per-channel partial sums:
 * actnn_batch_norm_workspace(N, C, HW) bytes for the current device, 16-byte aligned, its
 * contents need not be kept between calls.  Sums are added in a fixed order, so equal
 * inputs give equal bits. */
int64_t actnn_batch_norm_workspace(int64_t N, int64_t C, int64_t HW);
int actnn_batch_norm_forward(const void* x, const float* weight, const float* bias,
                             float* running_mean, float* running_var, void* y, float* save_mean,
                             float* save_invstd, int64_t N, int64_t C, int64_t HW, double momentum,
                             double eps, int dtype, void* workspace, int64_t workspace_bytes,
                             actnn_stream_t stream);
int actnn_batch_norm_backward(const void* x, const void* grad_out, const float* weight,
                              const float* save_mean, const float* save_invstd, void* grad_in,
                              float* grad_weight, float* grad_bias, int64_t N, int64_t C, int64_t HW,
                              int dtype, void* workspace, int64_t workspace_bytes,
                              actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * The four halves of a batch norm whose statistics are combined across ranks in between.
 * Replace the ATen operators the reference's synchronised batch norm calls: batch_norm_stats
 * (actnn/actnn/ops.py:515), batch_norm_elemt (ops.py:554), batch_norm_backward_reduce
 * (ops.py:570-577) and batch_norm_backward_elemt (ops.py:594-603).  Same tensors and meanings as those
 * operators: `mean` / `invstd` are float32 [C]; `sum_dy` = sum of grad_out, `sum_dy_xmu` = sum of
 * grad_out * (x - mean), `grad_weight` = sum_dy_xmu * invstd (sum_dy doubles as grad_bias);
 * `counts` = float32 device array of every rank's elements per channel (summed on the device,
 * so no host read is needed).  y of actnn_batch_norm_forward may be
 * NULL (statistics only); that is what actnn_batch_norm_stats calls.  Workspace as above
 * (the element-wise halves use its first 16 * C bytes). */
int actnn_batch_norm_stats(const void* x, float* mean, float* invstd, int64_t N, int64_t C,
                           int64_t HW, double eps, int dtype, void* workspace,
                           int64_t workspace_bytes, actnn_stream_t stream);
int actnn_batch_norm_elemt(const void* x, const float* weight, const float* bias,
                           const float* mean, const float* invstd, void* y, int64_t N, int64_t C,
                           int64_t HW, int dtype, void* workspace, int64_t workspace_bytes,
                           actnn_stream_t stream);
int actnn_batch_norm_backward_reduce(const void* x, const void* grad_out, const float* weight,
                                     const float* mean, const float* invstd, float* sum_dy,
                                     float* sum_dy_xmu, float* grad_weight, int64_t N, int64_t C,
                                     int64_t HW, int dtype, void* workspace,
                                     int64_t workspace_bytes, actnn_stream_t stream);
int actnn_batch_norm_backward_elemt(const void* x, const void* grad_out, const float* weight,
                                    const float* mean, const float* invstd, const float* sum_dy,
                                    const float* sum_dy_xmu, const float* counts, int64_t n_counts,
                                    void* grad_in, int64_t N, int64_t C, int64_t HW, int dtype,
                                    void* workspace, int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * 8-bit codes of rows (tokens, or the output channels of a weight), one float32 scale a row:
 * a = max |x| of the row (at least 1e-30), scale = a * (1/127), code = rint(x * (127 * (1/a))), half to even,
 * each step one rounded fp32 operation.  A row with a NaN or an infinity decodes to NaN.
 * `codes`: rows `ld_codes` bytes apart, the least multiple of 16 that holds `cols`, zero behind the
 * end; rows of x are `ld_x` elements apart (vector loads where x is on 16 bytes and cols and ld_x are
 * multiples of 8).  actnn_row_decode writes code * scale, [rows, cols] contiguous.
 * The reference has no counterpart (its codes are per group of 256 with a minimum,
 * actnn/actnn/cpp_extension/quantization_cuda_kernel.cu:86-142). */
int actnn_row_codes(const void* x, int8_t* codes, float* scale, int64_t rows, int64_t cols, int64_t ld_x,
                    int64_t ld_codes, int dtype, actnn_stream_t stream);
int actnn_row_decode(const int8_t* codes, const float* scale, void* out, int64_t rows, int64_t cols,
                     int64_t ld_codes, int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Sums over the rows of x [rows, cols], contiguous, in float32 and rounded once to `dtype`: the gradient of a
 * linear layer's bias (grad_output.sum(0), actnn/actnn/ops.py:425).  Fixed order of summation; workspace of
 * actnn_column_sums_workspace bytes, 4-byte aligned. */
int actnn_column_sums_workspace(int64_t rows, int64_t cols, int64_t* bytes);
int actnn_column_sums(const void* x, void* out, int64_t rows, int64_t cols, int dtype, void* workspace,
                      int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * out[t, n] = (sum_k tokens[t, k] * weights[n, k]) * token_scale[t] * channel_scale[n] + bias[n]
 * on the integer tensor cores; the sum is exact (int32), out is [T, N] contiguous of `dtype`, rounded
 * once.  `bias` (of `dtype`) may be NULL.  Rows of codes start on 16 bytes: pointers and ld_* (bytes)
 * are multiples of 16, and what lies between K and ld is not read as data.  1 <= K <= 131072.
 * A block whose bounded wait runs out leaves its outputs unwritten, as do those that share its reduction, and counts
 * the event (actnn_bulk_wait_failures).  The reference has no counterpart (its layers compute in the
 * activation's type, actnn/actnn/ops.py:408-428). */
int actnn_int8_matmul(const int8_t* tokens, const float* token_scale, const int8_t* weights,
                      const float* channel_scale, const void* bias, void* out, int64_t T, int64_t N, int64_t K,
                      int64_t ld_tokens, int64_t ld_weights, int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * A linear layer on a weight kept as codes: x [T, K] of `dtype`, rows `ld_x` elements apart, is coded as by
 * actnn_row_codes and multiplied as by actnn_int8_matmul, with the same result.  One launch for one token of up to
 * 48640 values and for up to eight with K <= 4096 and T * K <= 16384; otherwise `workspace`, 16-byte aligned, takes
 * the codes: actnn_int8_linear_workspace bytes (0: may be NULL).  The reference has no counterpart
 * (actnn/actnn/ops.py:408-428 computes in the activation's type). */
int actnn_int8_linear_workspace(int64_t T, int64_t K, int64_t* bytes);
int actnn_int8_linear(const void* x, const int8_t* weights, const float* channel_scale, const void* bias, void* out,
                      int64_t T, int64_t N, int64_t K, int64_t ld_x, int64_t ld_weights, int dtype, void* workspace,
                      int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Activation functions whose backward pass reads an 8-bit copy of the input.  `kind`: 0 identity, 1 ReLU,
 * 2 SiLU, 3 GELU (erf), 4 GELU (tanh form).  x is [rows, cols]; with `gated` it is [rows, 2 * cols] and
 * y = f(x[:, :cols]) * x[:, cols:].  y and grad_y are [rows, cols]; all contiguous.
 * With b = ceil(rows * cols / 256): `codes` has 256 * b bytes (gated: twice that, the gate's first), `scale`
 * b values (gated: 2 * b); 256 consecutive elements share a scale, coded as in actnn_row_codes.  NULL codes
 * and scale: nothing is saved, and the backward pass reads x instead (x may be NULL when codes are given).
 * The form without gate wants x, y, grad_y and grad_x on 16 bytes.  The reference has no counterpart (of its
 * activation functions ReLU saves one bit, actnn/actnn/cpp_extension/quantization.cc:106-124). */
int actnn_act_forward(const void* x, void* y, int8_t* codes, float* scale, int64_t rows, int64_t cols, int gated,
                      int kind, int dtype, actnn_stream_t stream);
int actnn_act_backward(const void* grad_y, const void* x, const int8_t* codes, const float* scale, void* grad_x,
                       int64_t rows, int64_t cols, int gated, int kind, int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Group norm with an activation (`kind` as above) on channels-last data [N, S, C], G groups of C / G channels:
 * y = f((x - mean) * rstd * gamma + beta), statistics over S * C / G elements, biased variance.
 * `codes` [N, S, C] (NULL: not saved) are 127 steps either way of the middle of each (sample, group)'s range;
 * `stats` float32 [N, G, 4] = mean, rstd, middle, half of the range (NULL only without codes: inference).
 * The backward pass computes with the decoded input, or with x where codes are NULL.  gamma, beta float32 or
 * NULL; grad_gamma, grad_beta (float32, NULL: not wanted) are sums over samples and positions.  Results are
 * reproducible (fixed order of summation).  Workspace: 16-byte aligned, actnn_group_norm_workspace bytes.
 * The reference has no counterpart (its norms are batch norms, actnn/actnn/ops.py:444-500). */
int actnn_group_norm_workspace(int64_t N, int64_t S, int64_t C, int64_t G, int64_t* bytes);
int actnn_group_norm_forward(const void* x, const float* gamma, const float* beta, void* y, int8_t* codes,
                             float* stats, int64_t N, int64_t S, int64_t C, int64_t G, double eps, int kind,
                             int dtype, void* workspace, int64_t workspace_bytes, actnn_stream_t stream);
int actnn_group_norm_backward(const void* grad_y, const void* x, const int8_t* codes, const float* stats,
                              const float* gamma, const float* beta, void* grad_x, float* grad_gamma,
                              float* grad_beta, int64_t N, int64_t S, int64_t C, int64_t G, int kind, int dtype,
                              void* workspace, int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Codes in 8-bit floating point (e4m3) with a power-of-two scale for each block of 128.  Of a block, e is the least
 * integer, at least -126, with max |x| <= 448 * 2^e; a code is x * 2^-e rounded to e4m3, half to even.  What is not
 * finite takes no part in the maximum and is coded as NaN.  `scales` are bytes e + 127 in the order
 * [ceil(cols / 512)][ceil(rows / 128)][512]: of 128 rows and four blocks, that of row r and block j at
 * (r % 32) * 16 + (r / 32) * 4 + j; bytes of rows behind the last are not written.  Rows of codes are ld_codes bytes
 * apart, the least multiple of 16 that holds them, zero behind the end; rows of x ld_x elements.
 * actnn_fp8_row_codes: blocks of 128 consecutive elements of a row.
 * actnn_fp8_tile_codes: the same to `codes`, and to `codes_t` [cols, ld_codes_t] the transposed matrix in blocks of
 * 128 consecutive rows of x; with `square` both in blocks of 128 x 128.  Either may be NULL.  parts (NULL: not wanted)
 * [ceil(rows / 128), cols]: sums of the columns of 128 rows, which actnn_fp8_join_sums adds in a fixed order.
 * actnn_fp8_decode: code * 2^e, [rows, cols] contiguous.
 * Code and scale pointers are on 16 bytes.  The reference has no counterpart (its codes are per group of 256 with a
 * minimum, actnn/actnn/cpp_extension/quantization_cuda_kernel.cu:86-142). */
int actnn_fp8_row_codes(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, int64_t ld_x,
                        int64_t ld_codes, int dtype, actnn_stream_t stream);
int actnn_fp8_tile_codes(const void* x, uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t,
                         float* parts, int64_t rows, int64_t cols, int64_t ld_x, int64_t ld_codes, int64_t ld_codes_t,
                         int square, int dtype, actnn_stream_t stream);
int actnn_fp8_join_sums(const float* parts, void* out, int64_t runs, int64_t cols, int dtype, actnn_stream_t stream);
int actnn_fp8_decode(const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols,
                     int64_t ld_codes, int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * out[t, n] = sum_k tokens[t, k] * weights[n, k] + bias[n] of what the codes above stand for, summed in fp32 on the
 * tensor cores; out is [T, N] contiguous of `dtype`, rounded once.  `bias` (of `dtype`) may be NULL.  What lies between
 * K and ld is not read as data.  Reproducible for given sizes.  A block whose bounded wait runs out leaves its
 * outputs unwritten, as do those that share its reduction, and counts the event (actnn_bulk_wait_failures).
 * The reference has no counterpart (its layers compute in the activation's type, actnn/actnn/ops.py:408-428). */
int actnn_fp8_matmul(const uint8_t* tokens, const uint8_t* token_scales, const uint8_t* weights,
                     const uint8_t* weight_scales, const void* bias, void* out, int64_t T, int64_t N, int64_t K,
                     int64_t ld_tokens, int64_t ld_weights, int dtype, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * A linear layer on a weight kept as codes: x [T, K] of `dtype`, rows `ld_x` elements apart, is coded as by
 * actnn_fp8_row_codes and multiplied.  One launch for up to eight tokens whose codes fit a block's shared memory;
 * otherwise `workspace`, 16-byte aligned, takes the codes: actnn_fp8_linear_workspace bytes (0: may be NULL).  The sums of
 * the one launch are added in another order than those of the other.  The reference has no counterpart
 * (actnn/actnn/ops.py:408-428 computes in the activation's type). */
int actnn_fp8_linear_workspace(int64_t T, int64_t K, int64_t* bytes);
int actnn_fp8_linear(const void* x, const uint8_t* weights, const uint8_t* weight_scales, const void* bias, void* out,
                     int64_t T, int64_t N, int64_t K, int64_t ld_x, int64_t ld_weights, int dtype, void* workspace,
                     int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Dropout whose mask is never stored.  Element e has the 16-bit field e % 8 (words and halves upwards) of the
 * Philox4x32-10 output for counter e / 8 and key (seed, offset), as actnn_dropout_forward; it is kept where
 * field + 1 > 65536 p, and multiplied by 1 / (1 - p).  y = x after it; the gradient is the same call on grad_y.
 * `state` (device, on 16 bytes; NULL: the key of the arguments): seed and offset, read by the kernel, for
 * launches that are replayed.  x and y contiguous, on 16 bytes.  0 <= p < 1.
 * actnn_philox_state writes such a state, (*seed, *offset + more), all on the device.
 * The reference keeps a bit an element (actnn/actnn/cpp_extension/quantization.cc:128-148). */
int actnn_seeded_dropout(const void* x, void* y, int64_t numel, float p, int dtype, uint64_t seed, uint64_t offset,
                         const int64_t* state, actnn_stream_t stream);
int actnn_philox_state(const int64_t* seed, const int64_t* offset, uint64_t more, int64_t* state,
                       actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * The norms before and after a block with its gate and residual scale, on rows of C channels (1 to 32768):
 *   r = scale * x + gate * drop(norm(f) * post_weight + post_bias),   h = norm(r) * weight + bias
 * `layer` 0: norm(v) = v / sqrt(mean(v^2) + eps); 1: of v less its mean.  `post` 0: f is taken as it is.
 * `gate` [rows / gate_rows, C]; it and the parameters [C], of param_dtype and gate_dtype, may be NULL (ones,
 * zeros).  Dropout as above, of element row * C + channel; p = 0: none.  x, f, r, h [rows, C] of `dtype`.
 * codes_x, codes_f [rows, C] with scales [rows, ceil(C / 256)] (all four NULL: not saved): the inputs in 8 bits
 * as in actnn_row_codes, 256 channels of a row to a scale.  stats [rows, 4] on 16 bytes: mean and reciprocal
 * deviation of f, of r (NULL only without codes).
 * Backward: of the codes, or of x and f where those are NULL.  grad_r or grad_h may be NULL (zeros); gradients
 * that are not wanted are NULL.  Those of parameters and gate are sums over rows in a fixed order, float32,
 * rounded once.  Workspace: 16-byte aligned, actnn_residual_norm_workspace bytes.  Blocks that share a row (C above
 * 4096) wait for one another's sums within limits: a wait that runs out is counted (actnn_bulk_wait_failures), and
 * the gradients that waited are NaN, those of the run's later rows too.
 * The reference has no counterpart (its norms are batch norms, actnn/actnn/ops.py:444-500). */
int actnn_residual_norm_forward(const void* x, const void* f, const void* weight, const void* bias,
                                const void* post_weight, const void* post_bias, const void* gate, void* r, void* h,
                                int8_t* codes_x, int8_t* codes_f, float* scale_x, float* scale_f, float* stats,
                                int64_t rows, int64_t C, int64_t gate_rows, double scale, double eps, int layer,
                                int post, float p, int dtype, int param_dtype, int gate_dtype, uint64_t seed,
                                uint64_t offset, const int64_t* state, actnn_stream_t stream);
int actnn_residual_norm_workspace(int64_t rows, int64_t C, int64_t gate_rows, int gate_grad, int64_t* bytes);
int actnn_residual_norm_backward(const void* grad_r, const void* grad_h, const void* x, const void* f,
                                 const int8_t* codes_x, const int8_t* codes_f, const float* scale_x,
                                 const float* scale_f, const float* stats, const void* weight,
                                 const void* post_weight, const void* post_bias, const void* gate, void* grad_x,
                                 void* grad_f, void* grad_weight, void* grad_bias, void* grad_post_weight,
                                 void* grad_post_bias, void* grad_gate, int64_t rows, int64_t C, int64_t gate_rows,
                                 double scale, int layer, int post, float p, int dtype, int param_dtype,
                                 int gate_dtype, uint64_t seed, uint64_t offset, const int64_t* state,
                                 void* workspace, int64_t workspace_bytes, actnn_stream_t stream);

/* ------------------------------------------------------------------------------------
 * How many bulk-copy waits gave up on the current device since the library was loaded.
 * The opt-in staged pack kernels (environment ACTNN_STAGED_PACK=1) copy their inputs into
 * shared memory with the bulk-copy engine and bound every wait on the completion barrier;
 * a warp whose wait runs out stops and leaves its outputs unwritten.  Zero in every
 * healthy run; reading it synchronises with the device.  No counterpart in the reference. */
int actnn_bulk_wait_failures(uint32_t* count);

/* ------------------------------------------------------------------------------------
 * How many four-group bundles actnn_pack_mixed / actnn_compress_mixed met, on the current
 * device since the library was loaded, whose per-sample width was outside 1..8: nothing is
 * written for such a bundle (the widths live on the device, so the entry point itself cannot
 * refuse them without a synchronisation).  Zero in every healthy run; reading it synchronises
 * with the device.  The reference accepts any width its caller passes
 * (quantization_cuda_kernel.cu:94-142) and has no such check. */
int actnn_bad_width_bundles(uint32_t* count);

/* ------------------------------------------------------------------------------------
 * The rounding noise the pack kernels draw for (seed, offset) when `noise == NULL`,
 * written as a [numel] array of `dtype` indexed like the padded [N, G, 256] activation.
 * No counterpart in the reference (it draws cuRAND numbers it cannot replay); exists so
 * that a CPU oracle can be fed the identical noise. */
int actnn_noise_fill(void* noise, int64_t numel, int dtype, uint64_t seed, uint64_t offset,
                     actnn_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif  /* ACTNN_B200_H_ */
