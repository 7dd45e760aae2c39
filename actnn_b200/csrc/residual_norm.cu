// The norms around a residual branch: arguments, and the cut of the kernels of residual_norm.cuh.
#include <algorithm>
#include <mutex>

#include "residual_norm.cuh"

namespace actnn {
namespace {

constexpr uint32_t kLeastRun = 8;                      // rows

int rn_shape(RnArgs& a, int64_t rows, int64_t C, int64_t gate_rows) {
  if (rows < 0 || rows > 0x7fffffff || C < 1 || C > kRnMostC || gate_rows < 1 || (rows > 0 && rows % gate_rows != 0)) return ACTNN_ERR_SHAPE;
  a.rows = (uint32_t)rows;
  a.C = (int)C;
  a.blocks = (int)((C + kRnBlock - 1) / kRnBlock);
  a.inv_c = 1.f / (float)C;
  a.by_gate = make_fast_div((uint32_t)std::min<int64_t>(gate_rows, 0x7fffffff));
  return ACTNN_OK;
}

// The runs of rows, one for every block (or cluster) that is resident at a time.  `gate`: the gate's gradient is wanted, so that no run
// reaches over a unit's end unless it has whole ones.  Few long units are cut, many or short ones go together.
void rn_runs(RnArgs& a, bool gate) {
  a.cluster = 1;
  while (a.cluster * kRnMostThreads * 8 < a.C) a.cluster *= 2;
  a.unit_rows = gate ? a.by_gate.d : a.rows;
  a.units = a.rows / a.unit_rows;
  const uint32_t threads = a.cluster > 1 ? kRnMostThreads : (a.C + 255) / 256 * 32, sms = device_info().sm_count;
  const uint32_t wanted = std::max(1u, sms * (kRnMostThreads / threads) / a.cluster);
  a.units_of_run = a.runs_of_unit = 0;
  if (gate && a.units > 1 && (a.unit_rows < kLeastRun || a.units >= wanted)) {
    a.units_of_run = std::max((kLeastRun + a.unit_rows - 1) / a.unit_rows, (a.units + wanted - 1) / wanted);
    a.runs = (a.units + a.units_of_run - 1) / a.units_of_run;
    return;
  }
  a.runs_of_unit = std::max(1u, std::min((a.unit_rows + kLeastRun - 1) / kLeastRun, wanted / a.units));
  a.runs = a.runs_of_unit * a.units;
}
int64_t rn_workspace_bytes(const RnArgs& a) { return (int64_t)a.runs * 5 * a.C * (int64_t)sizeof(float); }

int rn_dispatch(const RnArgs& a, int dtype, RnWhat what, bool vec) {
  return dtype == ACTNN_F32 ? rn_run_f32(a, what, vec) : dtype == ACTNN_F16 ? rn_run_f16(a, what, vec) : rn_run_bf16(a, what, vec);
}
// Parameters and gate.  What is not given gets the address of a tensor that is: C values of its own type, should a load come before the
// branch that it stands under.
void rn_parameters(RnArgs& a, const void* w1, const void* b1, const void* w2, const void* b2, const void* gate, int pdtype, int gdtype, const void* readable) {
  for (const void* p : {w1, b1, w2, b2}) if (p) readable = p;
  auto one = [&](const void* p, int dtype) { return p ? RnParameter{p, dtype} : RnParameter{readable, -1}; };
  a.w1 = one(w1, pdtype), a.b1 = one(b1, pdtype), a.w2 = one(w2, pdtype), a.b2 = one(b2, pdtype), a.gate = one(gate, gdtype);
  a.pdtype = pdtype, a.gdtype = gdtype;
}
bool rn_dtype(int d) { return d >= ACTNN_F32 && d <= ACTNN_BF16; }

}  // namespace

// Asked of the occupancy calculator once for each kernel, number of threads and device (the shared memory follows from these).
int rn_blocks_per_sm(const void* kernel, int threads, int smem) {
  struct Entry { const void* kernel; int threads, device, blocks; };
  static Entry table[2048];
  static int used = 0;
  static std::mutex lock;
  int device = 0, blocks = 0;
  cudaGetDevice(&device);
  std::lock_guard<std::mutex> guard(lock);
  for (int i = 0; i < used; ++i)
    if (table[i].kernel == kernel && table[i].threads == threads && table[i].device == device) return table[i].blocks;
  // one limit for all sizes: what is left of an SM's 227 KB besides the kernel's own
  cudaFuncAttributes own{};
  if (cudaFuncGetAttributes(&own, kernel) == cudaSuccess)
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)own.sharedSizeBytes);
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, threads, smem) != cudaSuccess || blocks < 1) blocks = 1;
  cudaGetLastError();
  if (used < 2048) table[used++] = Entry{kernel, threads, device, blocks};
  return blocks;
}
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_residual_norm_forward(const void* x, const void* f, const void* weight, const void* bias, const void* post_weight,
                                           const void* post_bias, const void* gate, void* r, void* h, int8_t* codes_x, int8_t* codes_f,
                                           float* scale_x, float* scale_f, float* stats, int64_t rows, int64_t C, int64_t gate_rows,
                                           double scale, double eps, int layer, int post, float p, int dtype, int param_dtype,
                                           int gate_dtype, uint64_t seed, uint64_t offset, const int64_t* state, actnn_stream_t stream) {
  RnArgs a{};
  if (int st = rn_shape(a, rows, C, gate_rows)) return st;
  if (layer < 0 || layer > 1 || post < 0 || post > 1 || !(eps >= 0.0) || !(p >= 0.f && p < 1.f) || (!layer && (bias || post_bias)) ||
      (!post && (post_weight || post_bias))) return ACTNN_ERR_ARG;
  if (!rn_dtype(dtype) || !rn_dtype(param_dtype) || !rn_dtype(gate_dtype)) return ACTNN_ERR_DTYPE;
  if (rows == 0) return ACTNN_OK;
  if (!x || !f || !r || !h || (!codes_x != !codes_f) || (codes_x && (!scale_x || !scale_f || !stats))) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype), psize = dtype_size(param_dtype);
  for (const void* q : {x, f, (const void*)r, (const void*)h}) if (!aligned(q, size)) return ACTNN_ERR_ALIGN;
  for (const void* q : {weight, bias, post_weight, post_bias}) if (!aligned(q, psize)) return ACTNN_ERR_ALIGN;
  if (!aligned(gate, dtype_size(gate_dtype)) || !aligned(stats, 16) || !aligned(scale_x, 4) || !aligned(scale_f, 4) || !aligned(state, 16)) return ACTNN_ERR_ALIGN;
  a.x = x; a.f = f; a.r = r; a.h = h;
  rn_parameters(a, post_weight, post_bias, weight, bias, gate, param_dtype, gate_dtype, x);
  a.cx = codes_x; a.cf = codes_f; a.sx = scale_x; a.sf = scale_f; a.stats = (float4*)stats;
  a.scale = (float)scale; a.eps = (float)eps; a.layer = layer; a.post = post; a.dropped = p > 0.f;
  a.drop = make_drop_key(p, seed, offset, state);
  a.stream = (cudaStream_t)stream;
  bool vec = C % 8 == 0 && aligned(codes_x, 8) && aligned(codes_f, 8);
  for (const void* q : {x, f, (const void*)r, (const void*)h, weight, bias, post_weight, post_bias, gate}) vec = vec && aligned(q, 16);
  return rn_dispatch(a, dtype, kRnForward, vec);
}

extern "C" int actnn_residual_norm_workspace(int64_t rows, int64_t C, int64_t gate_rows, int gate_grad, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  RnArgs a{};
  if (int st = rn_shape(a, rows, C, gate_rows)) return st;
  *bytes = 256;
  if (rows == 0) return ACTNN_OK;
  rn_runs(a, gate_grad != 0);
  *bytes = rn_workspace_bytes(a);
  return ACTNN_OK;
}

extern "C" int actnn_residual_norm_backward(const void* grad_r, const void* grad_h, const void* x, const void* f, const int8_t* codes_x,
                                            const int8_t* codes_f, const float* scale_x, const float* scale_f, const float* stats,
                                            const void* weight, const void* post_weight, const void* post_bias, const void* gate,
                                            void* grad_x, void* grad_f, void* grad_weight, void* grad_bias, void* grad_post_weight,
                                            void* grad_post_bias, void* grad_gate, int64_t rows, int64_t C, int64_t gate_rows, double scale,
                                            int layer, int post, float p, int dtype, int param_dtype, int gate_dtype, uint64_t seed,
                                            uint64_t offset, const int64_t* state, void* workspace, int64_t workspace_bytes,
                                            actnn_stream_t stream) {
  RnArgs a{};
  if (int st = rn_shape(a, rows, C, gate_rows)) return st;
  if (layer < 0 || layer > 1 || post < 0 || post > 1 || !(p >= 0.f && p < 1.f) || (!post && (post_weight || post_bias || grad_post_weight || grad_post_bias)) ||
      (!layer && (post_bias || grad_bias || grad_post_bias))) return ACTNN_ERR_ARG;
  if (!rn_dtype(dtype) || !rn_dtype(param_dtype) || !rn_dtype(gate_dtype)) return ACTNN_ERR_DTYPE;
  const int size = dtype_size(dtype), psize = dtype_size(param_dtype), gsize = dtype_size(gate_dtype);
  void* grads[5] = {grad_weight, grad_bias, grad_post_weight, grad_post_bias, grad_gate};
  for (int i = 0; i < 5; ++i) if (!aligned(grads[i], i < 4 ? psize : gsize)) return ACTNN_ERR_ALIGN;
  if (rows == 0) {                                       // sums of nothing; a gate for no rows has no values
    for (int i = 0; i < 4; ++i)
      if (grads[i] && cudaMemsetAsync(grads[i], 0, C * psize, (cudaStream_t)stream) != cudaSuccess) return ACTNN_ERR_LAUNCH;
    return ACTNN_OK;
  }
  if (!stats || !workspace || (!codes_x != !codes_f) || (codes_x ? !scale_x || !scale_f : !x || !f)) return ACTNN_ERR_NULL;
  const void* io[6] = {grad_r, grad_h, codes_x ? nullptr : x, codes_x ? nullptr : f, grad_x, grad_f};
  for (const void* q : io) if (!aligned(q, size)) return ACTNN_ERR_ALIGN;
  for (const void* q : {weight, post_weight, post_bias}) if (!aligned(q, psize)) return ACTNN_ERR_ALIGN;
  if (!aligned(gate, gsize) || !aligned(stats, 16) || !aligned(scale_x, 4) || !aligned(scale_f, 4) || !aligned(state, 16) || !aligned(workspace, 16)) return ACTNN_ERR_ALIGN;
  a.dr = grad_r; a.dh = grad_h; a.x = x; a.f = f; a.cx = (int8_t*)codes_x; a.cf = (int8_t*)codes_f; a.sx = (float*)scale_x; a.sf = (float*)scale_f;
  rn_parameters(a, post_weight, post_bias, weight, nullptr, gate, param_dtype, gate_dtype, workspace);
  a.stats = (float4*)stats; a.dx = grad_x; a.df = grad_f;
  a.scale = (float)scale; a.layer = layer; a.post = post; a.dropped = p > 0.f;
  a.drop = make_drop_key(p, seed, offset, state);
  a.coded = codes_x != nullptr;
  a.stream = (cudaStream_t)stream;
  rn_runs(a, grad_gate != nullptr);
  if (workspace_bytes < rn_workspace_bytes(a)) return ACTNN_ERR_CAPACITY;
  a.dw2 = grad_weight; a.db2 = grad_bias; a.dw1 = grad_post_weight; a.db1 = grad_post_bias; a.dgate = grad_gate;
  int* const slot[5] = {&a.slot_w2, &a.slot_b2, &a.slot_w1, &a.slot_b1, &a.slot_gate};         // the gate's last
  for (int i = 0; i < 5; ++i) *slot[i] = grads[i] && (i < 4 || a.units_of_run == 0) ? a.slots++ : -1;
  a.parts = (float*)workspace;
  bool vec = C % 8 == 0 && aligned(codes_x, 8) && aligned(codes_f, 8);
  for (const void* q : io) vec = vec && aligned(q, 16);
  for (const void* q : {weight, post_weight, post_bias, gate}) vec = vec && aligned(q, 16);
  return rn_dispatch(a, dtype, kRnBackward, vec);
}
