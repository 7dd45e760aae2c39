// The host side of the hot entry points in C++: outputs are allocated, the Philox offset is drawn and the
// library is called without going through Python for each of them, and the mask-saving layers (ReLU,
// dropout, max pooling) are C++ autograd functions, so that their backward passes run without the interpreter.
//
// A training step of small layers is paced by the host: a bf16 / float16 layer makes about ten allocations and
// calls of 10 - 25 arguments in each direction.  Measured a pass, float16, forward + backward: batch norm of
// 128 x 256 x 14 x 14 217 -> 162 us (46 on the GPU), the bottleneck block at batch 256 2400 -> 2209, compress and
// decompress of 8 x 16 x 14 x 14 46 -> 37.
// The Python functions of actnn_b200.cpp_extension keep the checks and the argument forms; this file has no
// behaviour of its own.
#include <ATen/Functions.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/CUDAGeneratorImpl.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <climits>
#include <mutex>

#include "../../include/actnn_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int dtype_id(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return ACTNN_F32;
    case at::kHalf: return ACTNN_F16;
    case at::kBFloat16: return ACTNN_BF16;
    default: TORCH_CHECK(false, "actnn_b200: unsupported dtype ", c10::toString(t));
  }
}
void check(int status, const char* what) {
  TORCH_CHECK(status == ACTNN_OK, what, " failed: ", actnn_status_string(status), " (status " + std::to_string(status) + ")");
}
actnn_stream_t stream() { return (actnn_stream_t)at::cuda::getCurrentCUDAStream().stream(); }
void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

// (seed, offset) from torch's default generator of the current device; advances the offset by one call.
std::pair<uint64_t, uint64_t> next_philox() {
  auto gen = at::cuda::detail::getDefaultCUDAGenerator();
  std::lock_guard<std::mutex> lock(gen.mutex());
  const uint64_t seed = gen.current_seed(), offset = gen.get_offset();
  gen.set_offset(offset + 4);
  return {seed, offset};
}
Tensor make(at::IntArrayRef shape, at::ScalarType t, const Tensor& like) {
  return at::empty(shape, like.options().dtype(t).memory_format(std::nullopt).requires_grad(false));
}
OptTensor as_f32(const OptTensor& t) {
  if (!t.has_value() || !t->defined()) return std::nullopt;
  return t->to(at::kFloat).contiguous();
}
at::ScalarType stat_type(const Tensor& data, bool bf16) { return bf16 ? at::kBFloat16 : data.scalar_type(); }

// ---------------------------------------------------------------------------------------- codec
// (packed, bits, scale, min, C, word_offsets); features < 0: data is [n, g, gs], whole groups
py::tuple compress_mixed(const Tensor& data, int64_t n, int64_t g, int64_t gs, int64_t features, double target_bits,
                         int64_t initial_bits, double range_factor, double coeff, const OptTensor& grad_scale,
                         bool stochastic, bool bf16_stats, const OptTensor& mn_in, const OptTensor& mx_in,
                         const OptTensor& ticket) {
  c10::cuda::CUDAGuard guard(data.device());
  const auto st = stat_type(data, bf16_stats);
  const int dt = dtype_id(data.scalar_type()), sd = dtype_id(st);
  const int64_t total = std::min(initial_bits * n, std::max((int64_t)target_bits, n));      // what the greedy ends with
  Tensor packed = make({(total * g * gs + 31) / 32}, at::kInt, data);
  Tensor scale = make({n, g, 1}, st, data), mn = make({n, g, 1}, st, data);
  Tensor bits = make({n}, at::kInt, data), offsets = make({n + 1}, at::kLong, data), C = make({n}, at::kFloat, data);
  uint64_t seed = 0, offset = 0;
  if (stochastic) std::tie(seed, offset) = next_philox();
  auto* words = packed.data_ptr<int32_t>();
  if (mn_in.has_value()) {
    check(actnn_compress_mixed_prestat_kept(data.data_ptr(), ptr(mn_in), ptr(mx_in), words, scale.data_ptr(), mn.data_ptr(),
                                            bits.data_ptr<int32_t>(), offsets.data_ptr<int64_t>(), C.data_ptr<float>(),
                                            ptr(ticket), n, g, gs, dt, sd, (float)range_factor, (float)coeff,
                                            (const float*)ptr(grad_scale), (int)initial_bits, target_bits, stochastic,
                                            nullptr, seed, offset, stream()),
          "actnn_compress_mixed_prestat_kept");
  } else {
    const int64_t bytes = actnn_compress_mixed_workspace(n, g, dt);
    Tensor ws = make({std::max<int64_t>(bytes, 256)}, at::kByte, data);
    if (features < 0)
      check(actnn_compress_mixed(data.data_ptr(), words, scale.data_ptr(), mn.data_ptr(), bits.data_ptr<int32_t>(),
                                 offsets.data_ptr<int64_t>(), C.data_ptr<float>(), ws.data_ptr(), bytes, n, g, gs, dt, sd,
                                 (float)range_factor, (float)coeff, (const float*)ptr(grad_scale), (int)initial_bits,
                                 target_bits, stochastic, nullptr, seed, offset, stream()),
            "actnn_compress_mixed");
    else
      check(actnn_compress_mixed_samples(data.data_ptr(), words, scale.data_ptr(), mn.data_ptr(),
                                         bits.data_ptr<int32_t>(), offsets.data_ptr<int64_t>(), C.data_ptr<float>(),
                                         ws.data_ptr(), bytes, n, features, dt, sd, (float)range_factor, (float)coeff,
                                         (const float*)ptr(grad_scale), (int)initial_bits, target_bits, stochastic,
                                         nullptr, seed, offset, stream()),
            "actnn_compress_mixed_samples");
  }
  return py::make_tuple(packed, bits, scale, mn, C, offsets);
}

Tensor unpack_mixed(const Tensor& packed, const Tensor& bits, const Tensor& offsets, const Tensor& scale, const Tensor& mn,
                    const std::vector<int64_t>& shape, int64_t n, int64_t g, int64_t gs, int64_t features,
                    const Tensor& like_dtype_of, bool as_float) {
  c10::cuda::CUDAGuard guard(packed.device());
  Tensor out = make(shape, as_float ? at::kFloat : like_dtype_of.scalar_type(), packed);
  const int dt = dtype_id(out.scalar_type()), sd = dtype_id(scale.scalar_type());
  if (features < 0)
    check(actnn_unpack_mixed(packed.data_ptr<int32_t>(), bits.data_ptr<int32_t>(), offsets.data_ptr<int64_t>(),
                             scale.data_ptr(), mn.data_ptr(), out.data_ptr(), n, g, gs, dt, sd, stream()),
          "actnn_unpack_mixed");
  else
    check(actnn_unpack_mixed_samples(packed.data_ptr<int32_t>(), bits.data_ptr<int32_t>(), offsets.data_ptr<int64_t>(),
                                     scale.data_ptr(), mn.data_ptr(), out.data_ptr(), n, features, dt, sd, stream()),
          "actnn_unpack_mixed_samples");
  return out;
}

// (packed, scale, min)
py::tuple compress_single(const Tensor& data, int64_t bits, bool stochastic, bool bf16_stats, int64_t bytes) {
  c10::cuda::CUDAGuard guard(data.device());
  const int64_t n = data.size(0), g = data.size(1), gs = data.size(2);
  const auto st = stat_type(data, bf16_stats);
  Tensor packed = make({bytes}, at::kChar, data), scale = make({n, g, 1}, st, data), mn = make({n, g, 1}, st, data);
  uint64_t seed = 0, offset = 0;
  if (stochastic) std::tie(seed, offset) = next_philox();
  check(actnn_compress_single(data.data_ptr(), (int)bits, packed.data_ptr<int8_t>(), scale.data_ptr(), mn.data_ptr(), nullptr,
                              n, g, gs, dtype_id(data.scalar_type()), dtype_id(st), stochastic, nullptr, seed, offset,
                              stream()),
        "actnn_compress_single");
  return py::make_tuple(packed, scale, mn);
}

// ---------------------------------------------------------------------------------------- batch norm
// (group minima, group maxima, mean, invstd), or None for a geometry that is not covered; `out`: room for the last two
py::object batch_norm_stats_minimax(const Tensor& x, const OptTensor& running_mean, const OptTensor& running_var,
                                    double momentum, double eps, const OptTensor& out) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t N = x.size(0), C = x.size(1), HW = N && C ? x.numel() / N / C : 0;
  const int64_t bytes = actnn_batch_norm_stats_minimax_workspace(N, C, HW);
  if (bytes < 0) return py::none();
  TORCH_CHECK(!out.has_value() || (out->scalar_type() == at::kFloat && out->is_contiguous() && out->numel() >= 2 * C &&
                                   out->device() == x.device()),
              "batch_norm_stats_minimax: out must be a contiguous float32 tensor of >= 2*C elements");
  const auto t = x.scalar_type();
  Tensor mn = make({N, C * HW / 256, 1}, t, x), mx = make({N, C * HW / 256, 1}, t, x);
  const Tensor both = out.has_value() ? out->view(-1) : make({2 * C}, at::kFloat, x);
  Tensor mean = both.narrow(0, 0, C), invstd = both.narrow(0, C, C);
  Tensor ws = make({bytes}, at::kByte, x);
  check(actnn_batch_norm_stats_minimax(x.data_ptr(), mn.data_ptr(), mx.data_ptr(), nullptr, nullptr,
                                       (float*)ptr(running_mean), (float*)ptr(running_var), mean.data_ptr<float>(),
                                       invstd.data_ptr<float>(), N, C, HW, momentum, eps, dtype_id(t), ws.data_ptr(),
                                       bytes, stream()),
        "actnn_batch_norm_stats_minimax");
  return py::make_tuple(mn, mx, mean, invstd);
}

// (y, packed, bits, scale, min, mean, invstd, word_offsets), or None for a geometry that is not covered
py::object batch_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& running_mean,
                              const OptTensor& running_var, double momentum, double eps, int64_t target_bits,
                              int64_t initial_bits, double range_factor, bool stochastic, const OptTensor& gmn,
                              const OptTensor& gmx, const OptTensor& mean_in, const OptTensor& invstd_in,
                              const Tensor& ticket) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t N = x.size(0), C = x.size(1), F = x.numel() / N, HW = F / C, G = (F + 255) / 256;
  const int dt = dtype_id(x.scalar_type());
  int64_t bytes = 0;
  if (actnn_batch_norm_codes_workspace(N, C, HW, dt, &bytes) != ACTNN_OK) return py::none();
  const auto st = stat_type(x, x.scalar_type() == at::kFloat);
  const int64_t total = std::min(initial_bits * N, std::max(target_bits, N));
  const OptTensor w = as_f32(weight), b = as_f32(bias);
  Tensor y = at::empty_like(x), packed = make({total * G * 8}, at::kInt, x);
  Tensor scale = make({N, G, 1}, st, x), mn = make({N, G, 1}, st, x), bits = make({N}, at::kInt, x);
  Tensor offsets = make({N + 1}, at::kLong, x), sens = make({N}, at::kFloat, x);
  Tensor mean = mean_in.has_value() ? *mean_in : make({C}, at::kFloat, x);
  Tensor invstd = invstd_in.has_value() ? *invstd_in : make({C}, at::kFloat, x);
  Tensor ws = make({bytes}, at::kByte, x);
  uint64_t seed = 0, offset = 0;
  if (stochastic) std::tie(seed, offset) = next_philox();
  check(actnn_batch_norm_codes_forward(
            x.data_ptr(), ptr(gmn), ptr(gmx), (const float*)ptr(w), (const float*)ptr(b), (float*)ptr(running_mean),
            (float*)ptr(running_var), y.data_ptr(), mean.data_ptr<float>(), invstd.data_ptr<float>(),
            packed.data_ptr<int32_t>(), scale.data_ptr(), mn.data_ptr(), bits.data_ptr<int32_t>(),
            offsets.data_ptr<int64_t>(), sens.data_ptr<float>(), N, C, HW, momentum, eps, dt, dtype_id(st),
            (float)range_factor, (int)initial_bits, (double)target_bits, stochastic, seed, offset, ticket.data_ptr(),
            ws.data_ptr(), bytes, stream()),
        "actnn_batch_norm_codes_forward");
  return py::make_tuple(y, packed, bits, scale, mn, mean, invstd, offsets);
}

// (grad_input, grad_weight, grad_bias), the last two in float32; None for a geometry that is not covered
py::object batch_norm_backward(const Tensor& packed, const Tensor& bits, const Tensor& offsets, const Tensor& scale,
                               const Tensor& mn, const std::vector<int64_t>& shape, const Tensor& grad_out, bool as_float,
                               const OptTensor& weight, const Tensor& mean, const Tensor& invstd) {
  c10::cuda::CUDAGuard guard(packed.device());
  int64_t F = 1;
  for (size_t i = 1; i < shape.size(); ++i) F *= shape[i];
  const int64_t N = shape[0], C = shape[1], HW = F / C;
  const auto t = as_float ? at::kFloat : scale.scalar_type();
  const int dt = dtype_id(t);
  int64_t bytes = 0;
  if (actnn_batch_norm_codes_workspace(N, C, HW, dt, &bytes) != ACTNN_OK) return py::none();
  const Tensor dy = grad_out.contiguous().to(t);
  const OptTensor w = as_f32(weight);
  Tensor dx = make(shape, t, packed), dw = make({C}, at::kFloat, packed), db = make({C}, at::kFloat, packed);
  Tensor ws = make({bytes}, at::kByte, packed);
  check(actnn_batch_norm_codes_backward(packed.data_ptr<int32_t>(), bits.data_ptr<int32_t>(), offsets.data_ptr<int64_t>(),
                                        scale.data_ptr(), mn.data_ptr(), dy.data_ptr(), (const float*)ptr(w),
                                        mean.data_ptr<float>(), invstd.data_ptr<float>(), dx.data_ptr(),
                                        dw.data_ptr<float>(), db.data_ptr<float>(), N, C, HW, dt,
                                        dtype_id(scale.scalar_type()), ws.data_ptr(), bytes, stream()),
        "actnn_batch_norm_codes_backward");
  return py::make_tuple(dx, dw, db);
}

// ---------------------------------------------------------------------------------------- small helpers
Tensor transpose16(const Tensor& x, bool to_channels_last) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = x.size(0), c = x.size(1), hw = x.size(2) * x.size(3);
  Tensor out = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(
      to_channels_last ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous));
  check(actnn_transpose16(x.data_ptr(), out.data_ptr(), n, to_channels_last ? c : hw, to_channels_last ? hw : c, stream()),
        "actnn_transpose16");
  return out;
}

Tensor sample_sumsq(const Tensor& grad_in) {
  c10::cuda::CUDAGuard guard(grad_in.device());
  const Tensor grad = grad_in.contiguous();
  const int64_t n = grad.size(0);
  Tensor out = make({n}, at::kFloat, grad);
  check(actnn_sample_sumsq(grad.data_ptr(), out.data_ptr<float>(), n, grad.numel() / std::max<int64_t>(n, 1),
                           dtype_id(grad.scalar_type()), stream()),
        "actnn_sample_sumsq");
  return out;
}

// The mean of sample_sumsq over the samples (0-dimensional); at least one sample
Tensor mean_sample_sumsq(const Tensor& grad_in, const Tensor& ticket) {
  c10::cuda::CUDAGuard guard(grad_in.device());
  const Tensor grad = grad_in.contiguous();
  const int64_t n = grad.size(0);
  Tensor out = make({n}, at::kFloat, grad), mean = make({}, at::kFloat, grad);
  check(actnn_sample_sumsq_mean(grad.data_ptr(), out.data_ptr<float>(), mean.data_ptr<float>(), ticket.data_ptr(), n,
                                grad.numel() / n, dtype_id(grad.scalar_type()), stream()),
        "actnn_sample_sumsq_mean");
  return mean;
}

// A copy of a small device tensor on its way to the host: enqueued on the current stream when made, waited for (by the
// host, without the interpreter lock) in `wait`.
struct Readback {
  Tensor host;
  at::cuda::CUDAEvent copied;
  explicit Readback(const Tensor& t) {
    c10::cuda::CUDAGuard guard(t.device());
    host = t.to(at::TensorOptions().device(at::kCPU), /*non_blocking=*/true);        // pinned
    copied.record();
  }
  Tensor wait() {
    py::gil_scoped_release unlocked;
    copied.synchronize();
    return host;
  }
};

// ---------------------------------------------------------------------------------------- mask-saving layers
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor mask_like(const Tensor& x) { return make({(x.numel() + 31) / 32}, at::kInt, x); }

Tensor relu_backward(const Tensor& grad_in, const Tensor& mask) {
  c10::cuda::CUDAGuard guard(grad_in.device());
  const Tensor grad = grad_in.contiguous();
  Tensor out = at::empty_like(grad);
  check(actnn_relu_backward(grad.data_ptr(), mask.data_ptr<int32_t>(), out.data_ptr(), grad.numel(),
                            dtype_id(grad.scalar_type()), stream()),
        "actnn_relu_backward");
  return out;
}

// ---------------------------------------------------------------------------------------- token operators
constexpr const char* kNames[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};
int activation_kind(const std::string& name) {
  for (int i = 0; i < 5; ++i)
    if (name == kNames[i]) return i;
  TORCH_CHECK(false, "activation must be one of gelu, gelu_tanh, none, relu, silu, got '", name, "'");
}
void check_values(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor!");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "The type of ", name,
              " is not correct!");
}
bool on16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor on_16_bytes(const Tensor& t) {
  Tensor c = t.contiguous();
  return on16(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}
int64_t row_bytes(int64_t k) { return (k + 15) / 16 * 16; }

// A matrix of the rows of x and the elements between them; copied only where the rows do not lie evenly.
std::pair<Tensor, int64_t> as_rows(const Tensor& x) {
  const int64_t k = x.size(-1);
  if (x.dim() == 2 && (x.stride(1) == 1 || k == 1) && (x.size(0) <= 1 || x.stride(0) >= k)) return {x, x.size(0) > 1 ? x.stride(0) : k};
  return {x.contiguous(), k};
}
// The same for codes, whose rows start on 16 bytes.
std::pair<Tensor, int64_t> code_rows(const Tensor& codes) {
  const int64_t k = codes.size(-1);
  Tensor c = codes.dim() == 2 ? codes : codes.reshape({k ? codes.numel() / k : 0, k});
  int64_t ld = c.size(0) > 1 ? c.stride(0) : row_bytes(k);
  if ((c.stride(1) != 1 && k > 1) || ld % 16 || ld < k || !on16(c)) {
    ld = row_bytes(k);
    Tensor padded = at::zeros({c.size(0), ld}, c.options());
    padded.narrow(1, 0, k).copy_(c);
    c = padded.narrow(1, 0, k);
  }
  return {c, ld};
}
struct RowCodes { Tensor codes, scale; int64_t rows, k, ld; };       // codes: [rows, ld]
RowCodes row_codes(const Tensor& x) {
  const auto [flat, ldx] = as_rows(x);
  const int64_t k = x.size(-1), rows = k ? x.numel() / k : 0, ld = row_bytes(k);
  RowCodes r{make({rows, ld}, at::kChar, x), make({rows}, at::kFloat, x), rows, k, ld};
  check(actnn_row_codes(flat.data_ptr(), r.codes.data_ptr<int8_t>(), r.scale.data_ptr<float>(), rows, k, ldx, ld,
                        dtype_id(x.scalar_type()), stream()),
        "actnn_row_codes");
  return r;
}
Tensor row_decode(const RowCodes& r, at::ScalarType t) {
  Tensor out = make({r.rows, r.k}, t, r.codes);
  check(actnn_row_decode(r.codes.data_ptr<int8_t>(), r.scale.data_ptr<float>(), out.data_ptr(), r.rows, r.k, r.ld, dtype_id(t), stream()),
        "actnn_row_decode");
  return out;
}
// The sums over the rows of a matrix.
Tensor column_sums(const Tensor& x_in) {
  const Tensor x = x_in.contiguous();
  const int64_t rows = x.size(0), cols = x.size(1);
  Tensor out = make({cols}, x.scalar_type(), x);
  int64_t bytes = 0;
  check(actnn_column_sums_workspace(rows, cols, &bytes), "actnn_column_sums_workspace");
  Tensor ws = make({bytes}, at::kByte, x);
  check(actnn_column_sums(x.data_ptr(), out.data_ptr(), rows, cols, dtype_id(x.scalar_type()), ws.data_ptr(), bytes, stream()),
        "actnn_column_sums");
  return out;
}
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}
void check_bias(const OptTensor& bias, const Tensor& x, int64_t n) {
  if (!bias.has_value() || !bias->defined()) return;
  check_values(*bias, "bias");
  TORCH_CHECK(bias->device() == x.device(), "bias is on ", bias->device(), ", expected ", x.device());
  TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n, "The dimension of bias is not correct!");
}
constexpr int64_t kMostK = 131072;

Tensor int8_linear(const Tensor& x, const Tensor& codes, const Tensor& scale, const OptTensor& bias) {
  check_values(x, "x");
  TORCH_CHECK(codes.is_cuda(), "weight_codes must be a CUDA tensor!");
  TORCH_CHECK(codes.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat,
              "The type of weight_codes is not correct! (int8 codes, float32 scales)");
  TORCH_CHECK(codes.dim() == 2 && scale.dim() == 1 && scale.size(0) == codes.size(0), "The dimension of weight_codes is not correct!");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == codes.size(1), "shapes ", x.sizes(), " and ", codes.sizes(), " cannot be multiplied");
  const int64_t n = codes.size(0), k = codes.size(1);
  TORCH_CHECK(k <= kMostK, "a product over ", k, " values may overflow its 32-bit sum; at most ", kMostK, " are accepted");
  TORCH_CHECK(codes.device() == x.device() && scale.device() == x.device(), "the weight is on ", codes.device(), ", the tokens on ", x.device());
  check_bias(bias, x, n);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = make(with_last(x, n), x.scalar_type(), x);
  const bool with = bias.has_value() && bias->defined();
  const Tensor b = with ? bias->to(x.scalar_type()).contiguous() : Tensor();
  if (k == 0) return with ? out.copy_(b) : out.zero_();
  const auto [flat, ldx] = as_rows(x);
  const auto [w, ldw] = code_rows(codes);
  const Tensor s = scale.contiguous();
  const int64_t rows = x.numel() / k;
  int64_t bytes = 0;
  check(actnn_int8_linear_workspace(rows, k, &bytes), "actnn_int8_linear_workspace");
  Tensor ws;
  if (bytes) ws = make({bytes}, at::kByte, x);
  check(actnn_int8_linear(flat.data_ptr(), w.data_ptr<int8_t>(), s.data_ptr<float>(), with ? b.data_ptr() : nullptr, out.data_ptr(), rows, n,
                          k, ldx, ldw, dtype_id(x.scalar_type()), bytes ? ws.data_ptr() : nullptr, bytes, stream()),
        "actnn_int8_linear");
  return out;
}

// (y, codes, scale); the latter undefined unless `save`
std::tuple<Tensor, Tensor, Tensor> act_forward(const Tensor& x_in, int kind, bool gated, bool save) {
  check_values(x_in, "x");
  int64_t cols = x_in.dim() ? x_in.size(-1) : 1;
  TORCH_CHECK(!gated || (x_in.dim() >= 1 && cols % 2 == 0), "a gated activation splits its last dimension in two, got shape ", x_in.sizes());
  if (gated) cols /= 2;
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = on_16_bytes(x_in);
  Tensor y = gated ? make(with_last(x, cols), x.scalar_type(), x) : make(x.sizes(), x.scalar_type(), x), codes, scale;
  const int64_t blocks = (y.numel() + 255) / 256 * (gated ? 2 : 1);
  if (save) codes = make({blocks * 256}, at::kChar, x), scale = make({blocks}, at::kFloat, x);
  if (y.numel())
    check(actnn_act_forward(x.data_ptr(), y.data_ptr(), save ? codes.data_ptr<int8_t>() : nullptr, save ? scale.data_ptr<float>() : nullptr,
                            y.numel() / cols, cols, gated, kind, dtype_id(x.scalar_type()), stream()),
          "actnn_act_forward");
  return {y, codes, scale};
}
Tensor act_backward(const Tensor& grad, const Tensor& x_in, const Tensor& codes, const Tensor& scale, int kind, bool gated) {
  c10::cuda::CUDAGuard guard(grad.device());
  const Tensor dy = on_16_bytes(grad);
  const int64_t cols = dy.dim() ? dy.size(-1) : 1;
  Tensor x, out = gated ? make(with_last(dy, 2 * cols), dy.scalar_type(), dy) : make(dy.sizes(), dy.scalar_type(), dy);
  if (!codes.defined()) x = on_16_bytes(x_in);
  if (dy.numel())
    check(actnn_act_backward(dy.data_ptr(), x.defined() ? x.data_ptr() : nullptr, codes.defined() ? codes.data_ptr<int8_t>() : nullptr,
                             codes.defined() ? scale.data_ptr<float>() : nullptr, out.data_ptr(), dy.numel() / cols, cols, gated, kind,
                             dtype_id(dy.scalar_type()), stream()),
          "actnn_act_backward");
  return out;
}

// x as contiguous [N, ..., C]
Tensor channels_behind(const Tensor& x) { return x.movedim(1, -1).contiguous(); }
OptTensor norm_parameter(const OptTensor& p, const char* name, const Tensor& x) {
  if (!p.has_value() || !p->defined()) return std::nullopt;
  check_values(*p, name);
  TORCH_CHECK(p->device() == x.device(), name, " is on ", p->device(), ", expected ", x.device());
  TORCH_CHECK(p->dim() == 1 && p->size(0) == x.size(1), name, " must have one value for each of the ", x.size(1), " channels");
  return as_f32(p->detach());
}
Tensor norm_workspace(const Tensor& x, int64_t n, int64_t s, int64_t c, int64_t groups) {
  int64_t bytes = 0;
  check(actnn_group_norm_workspace(n, s, c, groups, &bytes), "actnn_group_norm_workspace");
  return make({bytes}, at::kByte, x);
}
struct NormForward { Tensor y, last, codes, stats; };
NormForward norm_forward(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps, int kind, bool codes,
                         bool stats) {
  check_values(x, "x");
  TORCH_CHECK(x.dim() >= 2, "The dimension of x is not correct!");
  const int64_t n = x.size(0), c = x.size(1);
  TORCH_CHECK(groups >= 1 && c >= 1 && c % groups == 0, c, " channels cannot be split into ", groups, " groups");
  c10::cuda::CUDAGuard guard(x.device());
  NormForward r;
  r.last = channels_behind(x);
  int64_t s = 1;
  for (int64_t i = 2; i < x.dim(); ++i) s *= x.size(i);
  const OptTensor w = norm_parameter(weight, "weight", x), b = norm_parameter(bias, "bias", x);
  Tensor y = make(r.last.sizes(), x.scalar_type(), x);
  if (codes) r.codes = make(r.last.sizes(), at::kChar, x);
  if (stats) r.stats = make({n, groups, 4}, at::kFloat, x);
  const Tensor ws = norm_workspace(x, n, s, c, groups);
  check(actnn_group_norm_forward(r.last.data_ptr(), (const float*)ptr(w), (const float*)ptr(b), y.data_ptr(),
                                 codes ? r.codes.data_ptr<int8_t>() : nullptr, stats ? r.stats.data_ptr<float>() : nullptr, n, s, c, groups,
                                 eps, kind, dtype_id(x.scalar_type()), ws.data_ptr(), ws.numel(), stream()),
        "actnn_group_norm_forward");
  r.y = y.movedim(-1, 1);
  return r;
}

// with_minmax: also min and max of every 256 outputs, not differentiable
struct Relu : torch::autograd::Function<Relu> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, bool with_minmax) {
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty_like(x), mask = mask_like(x);
    const int dt = dtype_id(x.scalar_type());
    variable_list out{y};
    if (with_minmax) {
      ctx->set_materialize_grads(false);               // no zero-filled gradients for the extrema; y's is filled below
      ctx->saved_data["sizes"] = x.sizes();
      ctx->saved_data["dtype"] = x.scalar_type();
      Tensor mn = make({x.numel() / 256}, x.scalar_type(), x), mx = make({x.numel() / 256}, x.scalar_type(), x);
      check(actnn_relu_forward_minimax(x.data_ptr(), y.data_ptr(), mask.data_ptr<int32_t>(), mn.data_ptr(), mx.data_ptr(),
                                       x.numel(), dt, stream()),
            "actnn_relu_forward_minimax");
      ctx->mark_non_differentiable({mn, mx});
      out.push_back(mn);
      out.push_back(mx);
    } else {
      check(actnn_relu_forward(x.data_ptr(), y.data_ptr(), mask.data_ptr<int32_t>(), x.numel(), dt, stream()),
            "actnn_relu_forward");
    }
    ctx->save_for_backward({mask});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor mask = ctx->get_saved_variables()[0];
    if (grads[0].defined()) return {relu_backward(grads[0], mask), Tensor()};
    // the layer above gave no gradient, which counts as zeros
    return {at::zeros(ctx->saved_data["sizes"].toIntVector(), mask.options().dtype(ctx->saved_data["dtype"].toScalarType())),
            Tensor()};
  }
};

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p) {
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty_like(x), mask = mask_like(x);
    const auto [seed, offset] = next_philox();
    check(actnn_dropout_forward(x.data_ptr(), y.data_ptr(), mask.data_ptr<int32_t>(), x.numel(), (float)p,
                                dtype_id(x.scalar_type()), nullptr, seed, offset, stream()),
          "actnn_dropout_forward");
    ctx->save_for_backward({mask});
    ctx->saved_data["p"] = p;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor grad = grads[0].contiguous(), mask = ctx->get_saved_variables()[0];
    c10::cuda::CUDAGuard guard(grad.device());
    Tensor out = at::empty_like(grad);
    check(actnn_dropout_backward(grad.data_ptr(), mask.data_ptr<int32_t>(), out.data_ptr(), grad.numel(),
                                 (float)ctx->saved_data["p"].toDouble(), dtype_id(grad.scalar_type()), stream()),
          "actnn_dropout_backward");
    return {out, Tensor()};
  }
};

struct MaxPool : torch::autograd::Function<MaxPool> {
  // geom: kernel, stride, padding, dilation, two values each
  static Tensor forward(AutogradContext* ctx, const Tensor& x, std::vector<int64_t> geom) {
    TORCH_CHECK(geom.size() == 8 && x.dim() == 4, "max_pool2d: a 4-dimensional input and eight geometry values are expected");
    int g[8];
    for (int i = 0; i < 8; ++i) {                      // the output size below divides by the stride
      const int64_t least = i == 4 || i == 5 ? 0 : 1;
      TORCH_CHECK(geom[i] >= least && geom[i] <= INT_MAX, "max_pool2d: kernel_size, stride and dilation must be positive and padding "
                  "not negative, got ", geom[i]);
      g[i] = (int)geom[i];
    }
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t n = x.size(0), c = x.size(1), h = x.size(2), w = x.size(3);
    auto floordiv = [](int64_t a, int64_t b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); };
    const int64_t ho = floordiv(h + 2 * g[4] - (int64_t)g[6] * (g[0] - 1) - 1, g[2]) + 1;
    const int64_t wo = floordiv(w + 2 * g[5] - (int64_t)g[7] * (g[1] - 1) - 1, g[3]) + 1;
    Tensor y = make({n, c, ho, wo}, x.scalar_type(), x), idx = make({n, c, ho, wo}, at::kChar, x);
    check(actnn_max_pool2d_forward(x.data_ptr(), y.data_ptr(), idx.data_ptr<int8_t>(), n, c, h, w, g[0], g[1], g[2], g[3],
                                   g[4], g[5], g[6], g[7], dtype_id(x.scalar_type()), stream()),
          "actnn_max_pool2d_forward");
    ctx->save_for_backward({idx});
    ctx->saved_data["geom"] = geom;
    ctx->saved_data["shape"] = std::vector<int64_t>{n, c, h, w};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor grad = grads[0].contiguous(), idx = ctx->get_saved_variables()[0];
    c10::cuda::CUDAGuard guard(grad.device());
    const auto g = ctx->saved_data["geom"].toIntVector(), s = ctx->saved_data["shape"].toIntVector();
    Tensor out = make(s, grad.scalar_type(), grad);
    check(actnn_max_pool2d_backward(grad.data_ptr(), idx.data_ptr<int8_t>(), out.data_ptr(), s[0], s[1], s[2], s[3],
                                    (int)g[0], (int)g[1], (int)g[2], (int)g[3], (int)g[4], (int)g[5], (int)g[6], (int)g[7],
                                    dtype_id(grad.scalar_type()), stream()),
          "actnn_max_pool2d_backward");
    return {out, Tensor()};
  }
};

// x, weight, bias -> x weight^T + bias in 8-bit integers; the codes of both operands are kept
struct Int8Linear : torch::autograd::Function<Int8Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    check_values(x, "x");
    check_values(weight, "weight");
    TORCH_CHECK(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1), "shapes ", x.sizes(), " and ", weight.sizes(),
                " cannot be multiplied");
    TORCH_CHECK(weight.device() == x.device(), "the weight is on ", weight.device(), ", the tokens on ", x.device());
    const int64_t n = weight.size(0), k = weight.size(1);
    TORCH_CHECK(k <= kMostK, "a product over ", k, " values may overflow its 32-bit sum; at most ", kMostK, " are accepted");
    check_bias(bias, x, n);
    const bool with = bias.has_value() && bias->defined();
    c10::cuda::CUDAGuard guard(x.device());
    const RowCodes cx = row_codes(x), cw = row_codes(weight);
    Tensor out = make(with_last(x, n), x.scalar_type(), x);
    const Tensor b = with ? bias->to(x.scalar_type()).contiguous() : Tensor();
    if (k == 0)
      with ? out.copy_(b) : out.zero_();
    else
      check(actnn_int8_matmul(cx.codes.data_ptr<int8_t>(), cx.scale.data_ptr<float>(), cw.codes.data_ptr<int8_t>(), cw.scale.data_ptr<float>(),
                              with ? b.data_ptr() : nullptr, out.data_ptr(), cx.rows, n, k, cx.ld, cw.ld, dtype_id(x.scalar_type()), stream()),
            "actnn_int8_matmul");
    // the input's codes are what the weight's gradient is made of, and the other way round: what no gradient needs is not kept
    const bool keep_x = weight.requires_grad(), keep_w = x.requires_grad();
    ctx->save_for_backward({keep_x ? cx.codes : Tensor(), keep_x ? cx.scale : Tensor(), keep_w ? cw.codes : Tensor(),
                            keep_w ? cw.scale : Tensor()});
    ctx->saved_data["sizes"] = x.sizes();
    ctx->saved_data["n"] = n;
    ctx->saved_data["x"] = x.scalar_type();
    ctx->saved_data["w"] = weight.scalar_type();
    ctx->saved_data["b"] = with ? (int64_t)bias->scalar_type() : (int64_t)-1;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t k = sizes.back(), n = ctx->saved_data["n"].toInt();
    const auto type = ctx->saved_data["x"].toScalarType();
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) rows *= sizes[i];
    c10::cuda::CUDAGuard guard(grads[0].device());
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::AutocastCUDA);       // products in the types of the forward pass
    const Tensor go = grads[0].reshape({rows, n});
    Tensor gx, gw, gb;
    // The decoded operand of each product is rounded to the activation's type, as the operands of any layer in that type are; the
    // products' sums are float32.  bfloat16, 8192 x 2048 x 4096: the gradients are 0.0024 of their norm from the exact ones, of which
    // 0.0017 is their own rounding.  Products of the upper and of the lower half of each decoded value, added in float32,
    // leave 0.0017 and take 380 us instead of 190.
    if (ctx->needs_input_grad(0))
      gx = k ? go.mm(row_decode({saved[2], saved[3], n, k, row_bytes(k)}, type)).view(sizes) : at::zeros(sizes, go.options());
    if (ctx->needs_input_grad(1))
      gw = k ? go.t().mm(row_decode({saved[0], saved[1], rows, k, row_bytes(k)}, type)).to(ctx->saved_data["w"].toScalarType())
             : at::zeros({n, k}, go.options().dtype(ctx->saved_data["w"].toScalarType()));
    const int64_t bias_type = ctx->saved_data["b"].toInt();
    if (bias_type >= 0 && ctx->needs_input_grad(2)) gb = column_sums(go).to((at::ScalarType)bias_type);
    return {gx, gw, gb};
  }
};

// `compress` false: the input itself is kept.  The identity without a gate keeps nothing.
struct Activation : torch::autograd::Function<Activation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t kind, bool gated, bool compress) {
    const bool identity = kind == 0 && !gated;
    auto [y, codes, scale] = act_forward(x, (int)kind, gated, compress && !identity);
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["gated"] = gated;
    ctx->saved_data["compress"] = compress;
    if (compress && !identity) ctx->save_for_backward({codes, scale});
    else if (!identity) ctx->save_for_backward({x});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (saved.empty()) return {grads[0], Tensor(), Tensor(), Tensor()};
    const bool compress = ctx->saved_data["compress"].toBool();
    return {act_backward(grads[0], compress ? Tensor() : saved[0], compress ? saved[0] : Tensor(), compress ? saved[1] : Tensor(),
                         (int)ctx->saved_data["kind"].toInt(), ctx->saved_data["gated"].toBool()),
            Tensor(), Tensor(), Tensor()};
  }
};

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps,
                        int64_t kind, bool compress) {
    NormForward r = norm_forward(x, groups, weight, bias, eps, (int)kind, compress, true);
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["compress"] = compress;
    ctx->save_for_backward({compress ? r.codes : x, r.stats, weight.has_value() ? *weight : Tensor(), bias.has_value() ? *bias : Tensor()});
    return r.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool compress = ctx->saved_data["compress"].toBool();
    const Tensor &weight = saved[2], &bias = saved[3];
    const Tensor dy = grads[0];
    c10::cuda::CUDAGuard guard(dy.device());
    const Tensor last = channels_behind(dy), x = compress ? Tensor() : channels_behind(saved[0]);
    const int64_t n = dy.size(0), c = dy.size(1), groups = ctx->saved_data["groups"].toInt();
    int64_t s = 1;
    for (int64_t i = 2; i < dy.dim(); ++i) s *= dy.size(i);
    const OptTensor w = as_f32(weight), b = as_f32(bias);
    Tensor gx = make(last.sizes(), last.scalar_type(), last), gw, gb;
    if (weight.defined() && ctx->needs_input_grad(1)) gw = make({c}, at::kFloat, last);                    // counted without absent ones
    if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) gb = make({c}, at::kFloat, last);
    const Tensor ws = norm_workspace(last, n, s, c, groups);
    check(actnn_group_norm_backward(last.data_ptr(), compress ? nullptr : x.data_ptr(), compress ? saved[0].data_ptr<int8_t>() : nullptr,
                                    saved[1].data_ptr<float>(), (const float*)ptr(w), (const float*)ptr(b), gx.data_ptr(),
                                    gw.defined() ? gw.data_ptr<float>() : nullptr, gb.defined() ? gb.data_ptr<float>() : nullptr, n, s, c,
                                    groups, (int)ctx->saved_data["kind"].toInt(), dtype_id(last.scalar_type()), ws.data_ptr(), ws.numel(),
                                    stream()),
          "actnn_group_norm_backward");
    if (gw.defined()) gw = gw.to(weight.scalar_type());
    if (gb.defined()) gb = gb.to(bias.scalar_type());
    return {gx.movedim(-1, 1), Tensor(), gw, gb, Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::class_<Readback>(m, "Readback").def(py::init<const Tensor&>()).def("wait", &Readback::wait);
  m.def("compress_mixed", &compress_mixed);
  m.def("unpack_mixed", &unpack_mixed);
  m.def("compress_single", &compress_single);
  m.def("batch_norm_stats_minimax", &batch_norm_stats_minimax);
  m.def("batch_norm_forward", &batch_norm_forward);
  m.def("batch_norm_backward", &batch_norm_backward);
  m.def("transpose16", &transpose16);
  m.def("sample_sumsq", &sample_sumsq);
  m.def("mean_sample_sumsq", &mean_sample_sumsq);
  m.def("int8_linear", &int8_linear);
  m.def("int8_linear_train", [](const Tensor& x, const Tensor& w, const OptTensor& b) { return Int8Linear::apply(x, w, b); });
  m.def("activation", [](const Tensor& x, const std::string& name, bool gated, bool compress) {
    return Activation::apply(x, activation_kind(name), gated, compress);
  });
  m.def("group_norm", [](const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps, const std::string& name,
                         bool compress) { return GroupNorm::apply(x, groups, w, b, eps, activation_kind(name), compress); });
  m.def("group_norm_value", [](const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps,
                               const std::string& name) {
    return norm_forward(x, groups, w, b, eps, activation_kind(name), false, false).y;
  });
  m.def("relu", [](const Tensor& x) { return Relu::apply(x, false)[0]; });
  m.def("relu_minmax", [](const Tensor& x) { return Relu::apply(x, true); });
  m.def("dropout", [](const Tensor& x, double p) { return Dropout::apply(x, p); });
  m.def("max_pool2d", [](const Tensor& x, std::vector<int64_t> geom) { return MaxPool::apply(x, std::move(geom)); });
}
