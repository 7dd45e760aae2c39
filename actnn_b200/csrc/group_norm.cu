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
// The most runs of positions that two launches use: kGnFew positions a thread, kGnBlocks blocks for every SM.
constexpr int kGnFew = 4, kGnBlocks = 16;
int64_t most_runs(const GnShape& g, int64_t N) {
  const int64_t few = (int64_t)(kGnThreads / (g.tile / g.V)) * kGnFew, blocks = (int64_t)device_info().sm_count * kGnBlocks;
  return std::max<int64_t>(1, std::min((g.S + few - 1) / few, (blocks + N * g.tiles - 1) / (N * g.tiles)));
}

// One launch, where all its blocks fit the GPU at once (more of them run in step: all copy while the SMs idle, then all compute
// while the memory does.  Measured both ways, forward / backward in us, float16: 32 x 256 x 28 x 28 12.9 / 23.9 against 21.9 / 26.4
// of two launches, 1 x 256 x 64 x 64 11.0 / 15.4 against 16.9 / 54, but 256 x 256 x 28 x 28 68 / 125 against 68 / 99).
// Runs of channels of whole groups as narrow as still gives segments of kGnSegment bytes (they need no joining), then as many
// blocks in a cluster as it takes to hold the positions.  `size`: bytes of an element of the streamed tensor, `kept`: of what is
// kept of the input (0 in the forward pass).
constexpr int kGnSegment = 128, kGnCluster = 8;
bool hold_positions(GnShape& g, int64_t N, int size, int kept) {
  const int V = g.V;
  if (V < 2 || V * size < 4 || (kept > 0 && V * kept < 4)) return false;   // what the asynchronous copy does not know
  const int64_t sms = device_info().sm_count, whole = (int64_t)g.cpg / gcd(g.cpg, V) * V;
  for (const int segment : {kGnSegment, kGnSegment / 2}) {
    GnShape h = g;
    int64_t units = (segment + whole * size - 1) / (whole * size);
    if (units * whole > g.C) units = g.C / whole;
    h.tile = (int)(units * whole);
    h.parts = 1;
    if (units * whole > (int64_t)kGnThreads * V) continue;
    h.tiles = (g.C + h.tile - 1) / h.tile;
    const int R = kGnThreads / (h.tile / V), place = kGnThreads * V * (size + kept);
    for (int k = 1; k <= kGnCluster; k *= 2) {
      h.rows = (g.S + k - 1) / k;
      const int64_t held = (h.rows + R - 1) / R;
      if (held > kGnMostSmem / place) continue;
      const int64_t smem = gn_tables(h) + gn_scratch(h, kept == 0) + held * place;
      const int64_t resident = sms * std::min<int64_t>(size == 2 ? 3 : 2, (227 * 1024) / (smem + 1024));
      if (smem > kGnMostSmem || N * h.tiles * k > resident) continue;
      // more blocks while SMs are without one and a thread keeps kGnFew positions, while half of them are and it keeps one
      // (forward / backward, float16: 1 x 64 x 14 x 14 by one block 7.0 / 9.4 us, by four 6.4 / 7.9; 32 x 256 x 14 x 14 by 128 blocks
      // 7.7 / 10.2, by 256 9.2 / 11.4)
      const int64_t blocks = N * h.tiles * k, halved = g.S / (2 * k);
      if (k < kGnCluster && ((blocks < sms && halved >= (int64_t)R * kGnFew) || (2 * blocks < sms && halved >= R))) continue;
      h.chunks = k;
      h.held = (int)held;
      g = h;
      return true;
    }
  }
  return false;
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
// The widest vectors that the channels and the pointers take, and the cut of one launch where there is one.  `kept`: bytes of an
// element of what the backward pass reads of the input.
void gn_cut(GnShape& g, int64_t N, int dtype, const void* const* io, int n_io, const void* codes, int kept) {
  const int size = dtype_size(dtype);
  for (g.V = 16 / size; g.V > 1; g.V /= 2) {
    bool ok = aligned(codes, g.V);
    for (int i = 0; i < n_io; ++i) ok = ok && aligned(io[i], g.V * size);
    if (ok && cut_channels(g)) break;
  }
  cut_channels(g);                                       // one element a thread always fits
  if (!hold_positions(g, N, size, kept)) g.held = 0, g.chunks = 1;
  g.by_tiles = make_fast_div((uint32_t)g.tiles);
  g.by_chunks = make_fast_div((uint32_t)g.chunks);
  g.by_vecs = make_fast_div((uint32_t)(g.tile / g.V));
  g.by_cpg = make_fast_div((uint32_t)g.cpg);
  g.by_cells = make_fast_div((uint32_t)(g.cpg % g.V == 0 ? g.cpg / g.V : g.cpg));
}
// Most bytes that any cut needs: the partial statistics of two launches, and the sums of a backward pass (a cluster's blocks
// have them, too).
int64_t gn_bytes(GnShape g, int64_t N) {
  int64_t most = N * std::min<int64_t>(kGnCluster, g.S) * g.C * (int64_t)sizeof(float2);
  for (g.V = 8; g.V >= 1; g.V /= 2) {
    if (!cut_channels(g)) continue;
    const int64_t runs = most_runs(g, N);
    most = std::max(most, N * g.G * (runs * g.parts + 1) * (int64_t)sizeof(Part));               // and folded
    most = std::max(most, N * (runs + 1) * g.C * (int64_t)sizeof(float2));
  }
  return (most + 255) / 256 * 256;
}

}  // namespace

// Every launch ends with a wave that fills the GPU in part: the number of runs is the one for which the waves, each as long as a
// thread's positions and what a block does besides, are over first.
void gn_cut_positions(GnShape& g, int64_t N, int64_t resident, int extra) {
  const int R = kGnThreads / (g.tile / g.V);
  const int64_t most = most_runs(g, N);
  int64_t best = -1;
  for (int64_t k = 1; k <= most; ++k) {
    const int64_t rows = (g.S + k - 1) / k, time = (N * g.tiles * k + resident - 1) / resident * ((rows + R - 1) / R + extra);
    if (best >= 0 && time >= best) continue;
    best = time;
    g.rows = rows;
    g.chunks = (int)((g.S + rows - 1) / rows);
  }
  g.by_chunks = make_fast_div((uint32_t)g.chunks);
}

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
  g.wide = aligned(gamma, 16) && aligned(beta, 16);
  gn_cut(g, N, dtype, io, 2, codes, 0);
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
  g.wide = aligned(gamma, 16) && aligned(beta, 16);
  gn_cut(g, N, dtype, io, 3, codes, codes ? 1 : size);
  return dtype == ACTNN_F32 ? gn_run_f32(c, g, false) : dtype == ACTNN_F16 ? gn_run_f16(c, g, false) : gn_run_bf16(c, g, false);
}
