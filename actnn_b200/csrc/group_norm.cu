// Group norm with an activation, channels last: the float32 kernels, how the work is cut, and the C entry points.  The formulas
// and kernels are in group_norm.cuh.
#include <algorithm>

#include "group_norm.cuh"

namespace actnn {

int gn_run_f32(const GnCall& c, const GnShape& g, bool forward) { return gn_run<float>(c, g, forward); }

namespace {

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }
// Cuts the channels for vectors of g.V; false where they do not fit.
bool cut_channels(GnShape& g) {
  const int most = kGnThreads * g.V;
  if (g.C % g.V != 0) return false;
  const int64_t whole = (int64_t)g.cpg / gcd(g.cpg, g.V) * g.V;            // whole vectors of whole groups
  g.parts = 1;
  if (g.C <= most) {
    g.tile = g.C;
  } else if (whole <= most) {
    g.tile = (int)(most / whole * whole);
  } else {
    if (g.cpg % g.V != 0) return false;
    g.tile = most;
    g.parts = (g.cpg + most - 1) / most;
    g.tiles = g.G * g.parts;
    return true;
  }
  g.tiles = (g.C + g.tile - 1) / g.tile;
  return true;
}
// Runs of positions: as many blocks as keep the SMs supplied, but enough positions a thread that what a block does before and
// after them is little: kGnMany of them, or kGnFew until every SM has a block.
constexpr int kGnMany = 24, kGnFew = 4, kGnBlocks = 4;
void cut_positions(GnShape& g, int64_t N) {
  const int R = kGnThreads / (g.tile / g.V);
  const int64_t sms = device_info().sm_count, others = N * g.tiles;
  auto runs = [&](int64_t least) { return (g.S + R * least - 1) / (R * least); };
  auto fill = [&](int64_t blocks) { return (blocks + others - 1) / others; };
  int64_t k = std::max(std::min(runs(kGnMany), fill(sms * kGnBlocks)), std::min(runs(kGnFew), fill(sms)));
  if (k < 1) k = 1;
  g.rows = ((g.S + k - 1) / k + R - 1) / R * R;
  g.chunks = (int)((g.S + g.rows - 1) / g.rows);
}

int gn_shape(GnShape& g, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (N < 0 || S < 0 || C < 1 || G < 1 || C % G != 0 || C > (1 << 24)) return ACTNN_ERR_SHAPE;
  if (S > ((int64_t)1 << 38) / C || (N > 0 && S * C > ((int64_t)1 << 38) / N)) return ACTNN_ERR_SHAPE;     // more than memory holds
  g.S = S;
  g.C = (int)C;
  g.G = (int)G;
  g.cpg = (int)(C / G);
  return ACTNN_OK;
}
// The widest vectors that the channels and the pointers take; false where the grid would be too large.
bool gn_cut(GnShape& g, int64_t N, int dtype, const void* const* io, int n_io, const void* codes) {
  for (g.V = 8; g.V > 1; g.V /= 2) {
    const int bytes = g.V * dtype_size(dtype) < 16 ? g.V * dtype_size(dtype) : 16;
    bool ok = aligned(codes, g.V);
    for (int i = 0; i < n_io; ++i) ok = ok && aligned(io[i], bytes);
    if (ok && cut_channels(g)) break;
  }
  cut_channels(g);                                       // one element a thread always fits
  cut_positions(g, N);
  return N * g.chunks * g.tiles <= 0x7fffffff;
}
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
// Most bytes that any vector width needs.
int64_t gn_bytes(GnShape g, int64_t N) {
  int64_t most = 0;
  for (g.V = 8; g.V >= 1; g.V /= 2) {
    if (!cut_channels(g)) continue;
    cut_positions(g, N);
    const int64_t fwd = N * g.G * g.chunks * g.parts * (int64_t)sizeof(Part), bwd = N * g.chunks * g.C * (int64_t)sizeof(float2);
    most = fwd > most ? fwd : most;
    most = bwd > most ? bwd : most;
  }
  return align256(most);
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_group_norm_workspace(int64_t N, int64_t S, int64_t C, int64_t G, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  *bytes = N == 0 || S == 0 ? 256 : gn_bytes(g, N);
  return ACTNN_OK;
}

extern "C" int actnn_group_norm_forward(const void* x, const float* gamma, const float* beta, void* y, int8_t* codes, float* stats,
                                        int64_t N, int64_t S, int64_t C, int64_t G, double eps, int kind, int dtype,
                                        void* workspace, int64_t workspace_bytes, actnn_stream_t stream) {
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  if (kind < 0 || kind >= kActKinds || !(eps >= 0.0)) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (N == 0 || S == 0) return ACTNN_OK;
  if (!x || !y || !workspace || (codes && !stats)) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(x, size) || !aligned(y, size) || !aligned(workspace, 16) || !aligned(stats, 16)) return ACTNN_ERR_ALIGN;
  if (workspace_bytes < gn_bytes(g, N)) return ACTNN_ERR_CAPACITY;
  g.eps = (float)eps;
  const void* io[2] = {x, y};
  GnCall c{};
  c.x = x; c.gamma = gamma; c.beta = beta; c.out = y; c.codes = codes; c.stats = stats; c.workspace = workspace; c.N = N;
  c.kind = kind; c.stream = (cudaStream_t)stream;
  if (!gn_cut(g, N, dtype, io, 2, codes)) return ACTNN_ERR_SHAPE;
  return dtype == ACTNN_F32 ? gn_run_f32(c, g, true) : dtype == ACTNN_F16 ? gn_run_f16(c, g, true) : gn_run_bf16(c, g, true);
}

extern "C" int actnn_group_norm_backward(const void* grad_y, const void* x, const int8_t* codes, const float* stats,
                                         const float* gamma, const float* beta, void* grad_x, float* grad_gamma, float* grad_beta,
                                         int64_t N, int64_t S, int64_t C, int64_t G, int kind, int dtype, void* workspace,
                                         int64_t workspace_bytes, actnn_stream_t stream) {
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  if (kind < 0 || kind >= kActKinds) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (N == 0 || S == 0) {                                  // the gradients of the parameters are sums of nothing
    for (float* p : {grad_gamma, grad_beta})
      if (p && cudaMemsetAsync(p, 0, C * sizeof(float), (cudaStream_t)stream) != cudaSuccess) return ACTNN_ERR_LAUNCH;
    return ACTNN_OK;
  }
  if (!grad_y || !grad_x || !stats || !workspace || (!x && !codes)) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(grad_y, size) || !aligned(grad_x, size) || !aligned(workspace, 16) || !aligned(stats, 16)) return ACTNN_ERR_ALIGN;
  if (!codes && !aligned(x, size)) return ACTNN_ERR_ALIGN;
  if (workspace_bytes < gn_bytes(g, N)) return ACTNN_ERR_CAPACITY;
  const void* io[3] = {grad_y, grad_x, codes ? grad_y : x};
  GnCall c{};
  c.x = x; c.dy = grad_y; c.gamma = gamma; c.beta = beta; c.out = grad_x; c.codes = (int8_t*)codes; c.stats = (float*)stats;
  c.dgamma = grad_gamma; c.dbeta = grad_beta; c.workspace = workspace; c.N = N; c.kind = kind; c.stream = (cudaStream_t)stream;
  if (!gn_cut(g, N, dtype, io, 3, codes)) return ACTNN_ERR_SHAPE;
  return dtype == ACTNN_F32 ? gn_run_f32(c, g, false) : dtype == ACTNN_F16 ? gn_run_f16(c, g, false) : gn_run_bf16(c, g, false);
}
