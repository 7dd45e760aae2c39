// Matrix product of 8-bit integers with a scale for each token and each output channel:
//
//   out[t, n] = (sum_k x[t, k] * w[n, k]) * token_scale[t] * channel_scale[n] + bias[n]
//
// The sum is exact (int32; k <= 131072 keeps it below 2^31), the scales and the bias are applied in fp32 and rounded once.
//
// The tensor cores compute tiles of 128 channels (the rows of the accumulator, one lane of tensor memory each) by up to 256
// tokens (its columns): the operand with 128 rows is the weight, so that few tokens waste no work, and a thread of the
// epilogue has one channel, whose scale and bias stay in registers while 32 lanes write 32 neighbouring outputs of a token.
// A block is a pipeline: one thread requests tiles of both operands (128 bytes of the reduction a stage, swizzled for the
// matrix instructions), one issues the matrix instructions, eight warps scale and write one accumulator while the next one
// fills.  Where the tiles are too few for the SMs, the reduction is split over the blocks of a cluster, which add their
// integer sums through distributed shared memory: order does not matter to them.
//
// Where the tiles fill the GPU, two blocks compute one of 256 channels together: each loads half of the channels' operand and half
// of the tokens'.  Outputs are turned into rows of channels in shared memory and leave as boxes of 128 channels, because 32
// lanes' 64 bytes each took longer than the multiplication (8192 x 2048 x 4096: 87 us with them, 65 with boxes).
//
// Measured on a B200, bfloat16 outputs: 16384 x 4096 x 8192 340 - 360 us, 3.1e15 operations a second (twice the measured bfloat16 rate
// is 3.24e15; the tensor pipe is 79 - 82 % busy, the rest is the L2's, 12 TB/s); 8192 x 2048 x 4096 48 - 61; 200 x 4096 x 4096 12.5, where
// the weight's bytes take 2.6 and the fixed latencies of launch, first copies, sums through the cluster and outputs about 8.
//
// Every wait is bounded.  A block whose wait runs out writes nothing more, is counted (the counter of the bulk waits), lets
// its copies and instructions end and leaves.  The epilogue's warps leave together: its barriers count all of them.
#include <atomic>

#include "activation.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace actnn {
namespace {

constexpr int kMmThreads = 320;                 // 8 epilogue warps, one for the copies, one for the matrix instructions
constexpr int kMmEpilogue = 256;
constexpr int kMmStagesMost = 8, kMmSplitsMost = 8;
constexpr int kMmStageK = 128;                  // bytes of the reduction in a stage
constexpr int kMmChannels = 128;
constexpr int kMmStaging = 32 * 1024;           // outputs on their way: two buffers for each half of the epilogue's warps
constexpr int kMmSmem = 212 * 1024;             // of the SM's 227 KB: stages, and 1 KB to align them

struct MmArgs {
  const float *token_scale, *channel_scale;
  const void* bias;
  void* out;
  int64_t T, N;
  int K, tokens, stages, k_blocks, splits;      // tokens: columns of a tile
  int channel_tiles, tiles, columns;            // columns: of tensor memory, a buffer
  bool pair;                                    // tiles of 256 channels by pairs of blocks
  bool boxes;                                   // outputs leave as boxes of 128 channels
  bool vectors;                                 // four outputs of a token at a time are aligned
  bool early;                                   // the launch before this one makes the tokens' codes, and is not waited for sooner than they are read
};

struct MmShared {
  uint64_t full[kMmStagesMost], empty[kMmStagesMost], sum_full[2], sum_empty[2], drained;
  uint32_t tmem;
  int dead, gone;                               // a wait of the block has run out; of one of the blocks that share a reduction
  alignas(16) float scale[2][256];
};

// Tokens of a box: 8 KB of 128 channels.
template <typename T> constexpr int box_tokens() { return kMmStaging / 4 / (kMmChannels * (int)sizeof(T)); }
ACTNN_DEV void store_shared(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" :: "r"(at), "f"(v) : "memory"); }
ACTNN_DEV void store_shared(uint32_t at, __half v) { asm volatile("st.shared.u16 [%0], %1;" :: "r"(at), "h"(__half_as_ushort(v)) : "memory"); }
ACTNN_DEV void store_shared(uint32_t at, __nv_bfloat16 v) {
  asm volatile("st.shared.u16 [%0], %1;" :: "r"(at), "h"(__bfloat16_as_ushort(v)) : "memory");
}

// Waits for a phase; false once this or another wait of the block has run out.
ACTNN_DEV bool mm_wait(uint32_t bar, uint32_t parity, MmShared& s, unsigned* gave_up) {
  volatile int* dead = &s.dead;
  for (uint32_t i = 0; i < kBulkWaitTries; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*dead) return false;
  }
  *dead = 1;
  if (gave_up) atomicAdd(gave_up, 1u);
  return false;
}

// Of the epilogue's eight warps: whether the waits of all of them came to their end.  A warp that left alone, because another
// wait had run out just before its own phase was complete, would leave those whose phase was to barriers it never comes to.
ACTNN_DEV bool epilogue_agrees(bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
               "barrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)ok) : "memory");
  return all != 0;
}

// SPLIT: the reduction is split over a cluster.  PAIR: a cluster of two blocks computes a tile of 256 channels, half of the channels
// and half of the tokens' operand in each; the first one issues the matrix instructions, its barriers count the copies of both.
template <typename T, bool SPLIT, bool PAIR>
__global__ void __launch_bounds__(kMmThreads, 1)
int8_matmul_kernel(const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap tokens,
                   const __grid_constant__ CUtensorMap outputs, const MmArgs a, unsigned* gave_up) {
  extern __shared__ uint8_t dynamic_s[];
  __shared__ MmShared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stage0 = (smem_addr(dynamic_s) + 1023u) & ~1023u;
  const uint32_t rank = SPLIT || PAIR ? cluster_rank() : 0, split = SPLIT ? rank : 0;
  const int load_tokens = PAIR ? a.tokens / 2 : a.tokens, tile_channels = PAIR ? 2 * kMmChannels : kMmChannels;
  const uint32_t a_bytes = kMmChannels * kMmStageK, stage_bytes = a_bytes + load_tokens * kMmStageK;
  const int k_first = SPLIT ? (int)((int64_t)split * a.k_blocks / a.splits) : 0;
  const int k_end = SPLIT ? (int)((int64_t)(split + 1) * a.k_blocks / a.splits) : a.k_blocks;
  const int first_tile = SPLIT ? blockIdx.x / a.splits : PAIR ? blockIdx.x / 2 : blockIdx.x;
  const int tile_step = SPLIT ? a.tiles : PAIR ? gridDim.x / 2 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(smem_addr(&s.full[i]), 1);
      mbar_init(smem_addr(&s.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&s.sum_full[i]), 1);
      mbar_init(smem_addr(&s.sum_empty[i]), (PAIR ? 2 : 1) * kMmEpilogue / 32);
    }
    mbar_init(smem_addr(&s.drained), 1);
    s.dead = s.gone = 0;
    mbar_init_fence();
  }
  const uint32_t columns = SPLIT ? a.columns : 2 * a.columns;
  if (warp == 9) tmem_alloc<PAIR>(smem_addr(&s.tmem), columns);
  tmem_fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();                           // both blocks have their barriers and their tensor memory
  if constexpr (SPLIT) cluster_arrive();                        // this block's flags are set
  tmem_fence_after_sync();
  const uint32_t tmem = s.tmem;

  int copy_stage = 0, issued = 0, ahead = 0;                    // of the copies' thread, to the end
  uint32_t copy_phase = 0;
  bool copied = true;
  if (warp == 8) {                                              // ---------------- copies
    if (lane == 0) {
      // Requests one operand of a stage; of a pair, the first block's barrier counts.
      auto request = [&](int stage, uint32_t offset, const CUtensorMap* map, int k, int row) {
        const uint32_t dst = stage0 + stage * stage_bytes + offset, bar = smem_addr(&s.full[stage]);
        if constexpr (PAIR) tile_load_pair(dst, map, k * kMmStageK, row, peer_addr(bar, 0));
        else tile_load(dst, map, k * kMmStageK, row, bar);
      };
      auto expect = [&](int stage) {
        if (!PAIR || rank == 0) mbar_expect_tx(smem_addr(&s.full[stage]), PAIR ? 2 * stage_bytes : stage_bytes);
      };
      if (a.early) {                                            // weights of the first stages before the tokens are there
        const int ct = first_tile % a.channel_tiles;
        for (ahead = 0; first_tile < a.tiles && ahead < a.stages && ahead < k_end - k_first; ++ahead) {
          expect(ahead);
          request(ahead, 0, &weights, k_first + ahead, ct * tile_channels + (int)rank * kMmChannels * PAIR);
        }
        grid_wait();
      }
      for (int tile = first_tile; copied && tile < a.tiles; tile += tile_step) {
        const int tt = tile / a.channel_tiles, ct = tile - tt * a.channel_tiles;
        for (int k = k_first; k < k_end; ++k) {
          if (!(copied = mm_wait(smem_addr(&s.empty[copy_stage]), copy_phase ^ 1, s, gave_up))) break;
          if (issued >= ahead) {
            expect(copy_stage);
            request(copy_stage, 0, &weights, k, ct * tile_channels + (int)rank * kMmChannels * PAIR);
          }
          request(copy_stage, a_bytes, &tokens, k, tt * a.tokens + (int)rank * load_tokens * PAIR);
          ++issued;
          if (++copy_stage == a.stages) copy_stage = 0, copy_phase ^= 1;
        }
      }
      // A pair's second block is there until what the first one's matrix instructions arrive at has been arrived at: the stages' barriers
      // and the one for the end.  (In their own block the thread that issues them waits for the end.)
      for (int i = 0, at = copy_stage; PAIR && copied && i < a.stages; ++i) {
        copied = mm_wait(smem_addr(&s.empty[at]), copy_phase ^ (at < copy_stage ? 0 : 1), s, gave_up);
        if (++at == a.stages) at = 0;
      }
      if (PAIR && copied) copied = mm_wait(smem_addr(&s.drained), 0, s, gave_up);
    }
  } else if (warp == 9) {                                       // ---------------- matrix instructions
    if (a.early) grid_wait();                                   // the limit of a wait is for copies, not for the launch before
    if (lane == 0 && (!PAIR || rank == 0)) {
      const uint32_t instruction = int8_instruction(tile_channels, a.tokens);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
        if (!(ok = mm_wait(smem_addr(&s.sum_empty[buf]), buf_phase ^ 1, s, gave_up))) break;
        tmem_fence_after_sync();
        const uint32_t d = tmem + buf * a.columns;
        for (int k = k_first; k < k_end; ++k) {
          if (!(ok = mm_wait(smem_addr(&s.full[stage]), phase, s, gave_up))) break;
          tmem_fence_after_sync();
          const uint32_t at = stage0 + stage * stage_bytes;
          const uint64_t da = rows128_descriptor(at), db = rows128_descriptor(at + a_bytes);
#pragma unroll
          for (int i = 0; i < kMmStageK / 32; ++i)              // 32 bytes further along the rows: 2 in units of 16 bytes
            mma_int8<PAIR>(d, da + 2 * i, db + 2 * i, instruction, k > k_first || i > 0);
          mma_commit<PAIR>(smem_addr(&s.empty[stage]));
          if (++stage == a.stages) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        mma_commit<PAIR>(smem_addr(&s.sum_full[buf]));
        if (++buf == 2) buf = 0, buf_phase ^= 1;
      }
      mma_commit<PAIR>(smem_addr(&s.drained));
      mbar_wait(smem_addr(&s.drained), 0);
    }
    __syncwarp();
  } else {                                                      // ---------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    if (a.early) grid_wait();
    int buf = 0, box_buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = first_tile; tile < a.tiles; tile += tile_step) {
      const int tt = tile / a.channel_tiles, ct = tile - tt * a.channel_tiles;
      const int64_t t0 = (int64_t)tt * a.tokens, n = (int64_t)ct * tile_channels + rank * kMmChannels * PAIR + quarter * 32 + lane;
      if constexpr (!SPLIT) {
        if ((int)threadIdx.x < a.tokens) s.scale[buf][threadIdx.x] = t0 + threadIdx.x < a.T ? __ldg(a.token_scale + t0 + threadIdx.x) : 0.f;
      }
      const float w = n < a.N ? __ldg(a.channel_scale + n) : 0.f;
      const float b = n < a.N && a.bias ? to_float(reinterpret_cast<const T*>(a.bias)[n]) : 0.f;
      // One warp waits for the sums, the others for its word: sleepers wake up to a microsecond apart.
      const bool ok = warp != 0 || mm_wait(smem_addr(&s.sum_full[buf]), buf_phase, s, lane == 0 ? gave_up : nullptr);
      tmem_fence_after_sync();
      tmem_fence_before_sync();
      if (!epilogue_agrees(ok)) break;                          // and the scales are there for all
      tmem_fence_after_sync();
      const uint32_t d = tmem + buf * a.columns + ((uint32_t)(quarter * 32) << 16);
      if (!SPLIT && a.boxes) {
        // The warps of a half turn kBoxTokens columns into rows of 128 channels in shared memory, which one thread sends off as a
        // box while the next ones are made.
        constexpr int kBoxTokens = box_tokens<T>();
        for (int c = half * kBoxTokens; c < a.tokens; c += 2 * kBoxTokens) {
          const uint32_t box = stage0 + a.stages * stage_bytes + (half * 2 + box_buf) * (kMmStaging / 4);
          if ((threadIdx.x & 127) == 0) tile_store_read<1>();                       // the buffer's last box has been read
          asm volatile("bar.sync %0, 128;" :: "r"(2 + half) : "memory");
#pragma unroll
          for (int k = 0; k < kBoxTokens; k += 16) {
            uint32_t r[16];
            tmem_load16(d + c + k, r);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 q = *reinterpret_cast<const float4*>(&s.scale[buf][c + k + i]);
              const float sc[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                store_shared(box + ((k + i + j) * kMmChannels + quarter * 32 + lane) * sizeof(T),
                             from_float<T>(fmaf((float)(int)r[i + j] * sc[j], w, b)));
            }
          }
          tile_store_fence();
          asm volatile("bar.sync %0, 128;" :: "r"(2 + half) : "memory");
          if ((threadIdx.x & 127) == 0) tile_store(&outputs, (int)(n - lane), (int)(t0 + c), box);
          box_buf ^= 1;
        }
      } else
      for (int c = half * 16; c < a.tokens; c += 32) {
        uint32_t r[16];
        tmem_load16(d + c, r);
        tmem_load_wait();
        if constexpr (SPLIT) {                                  // [column][channel] over the stages, which are done with
          const uint32_t p = stage0 + c * (kMmChannels * 4) + (quarter * 32 + lane) * 4;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.u32 [%0], %1;" :: "r"(p + i * kMmChannels * 4), "r"(r[i]) : "memory");
        } else {
          T* o = reinterpret_cast<T*>(a.out) + (t0 + c) * a.N + n;
          const int left = (int)min((int64_t)16, a.T - t0 - c);
          if (n < a.N) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (i < left) o[i * a.N] = from_float<T>(fmaf((float)(int)r[i] * s.scale[buf][c + i], w, b));
          }
        }
      }
      if constexpr (!SPLIT) {
        tmem_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) peer_arrive(peer_addr(smem_addr(&s.sum_empty[buf]), 0));
          else mbar_arrive(smem_addr(&s.sum_empty[buf]));
        }
        if (++buf == 2) buf = 0, buf_phase ^= 1;
      }
    }
  }
  if (!SPLIT && a.boxes && warp < 8 && (threadIdx.x & 127) == 0) tile_store_done();
  if constexpr (SPLIT) {
    __syncwarp();
    cluster_wait();                                             // all have begun, long since
    // Where a wait of any of the cluster's blocks ran out, its sums are not there, and nothing is written by any of them.  The
    // thread whose wait it was has seen its block's flag set, and tells the others before it comes to the barrier.
    if (s.dead)
      for (int k = 0; k < a.splits; ++k) peer_store1(smem_addr(&s.gone), k, 1);
    cluster_sync();
    if (warp < 8 && !s.gone) {                                  // a warp takes a column: 4 channels a lane, all blocks' sums at once
      const int tt = first_tile / a.channel_tiles, ct = first_tile - tt * a.channel_tiles;
      const int64_t t0 = (int64_t)tt * a.tokens, n = (int64_t)ct * kMmChannels + lane * 4;
      float w[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = n + i < a.N ? __ldg(a.channel_scale + n + i) : 0.f;
        b[i] = n + i < a.N && a.bias ? to_float(reinterpret_cast<const T*>(a.bias)[n + i]) : 0.f;
      }
      const int end = (int)min((int64_t)a.tokens, a.T - t0);
#pragma unroll 2
      for (int c = (int)split + a.splits * warp; c < end; c += 8 * a.splits) {
        int4 part[kMmSplitsMost];
        const float scale = __ldg(a.token_scale + t0 + c);
#pragma unroll
        for (int k = 0; k < kMmSplitsMost; ++k)
          if (k < a.splits) part[k] = peer_load4i(stage0 + c * (kMmChannels * 4) + lane * 16, k);
        int4 sum = part[0];
#pragma unroll
        for (int k = 1; k < kMmSplitsMost; ++k)
          if (k < a.splits) sum.x += part[k].x, sum.y += part[k].y, sum.z += part[k].z, sum.w += part[k].w;
        float2 out[2] = {make_float2(fmaf((float)sum.x * scale, w[0], b[0]), fmaf((float)sum.y * scale, w[1], b[1])),
                         make_float2(fmaf((float)sum.z * scale, w[2], b[2]), fmaf((float)sum.w * scale, w[3], b[3]))};
        T* o = reinterpret_cast<T*>(a.out) + (t0 + c) * a.N + n;
        if (a.vectors && n + 4 <= a.N) {
          store_vec<T, 4>(o, out);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < a.N) o[i] = from_float<T>(i & 1 ? out[i / 2].y : out[i / 2].x);
        }
      }
    }
    cluster_sync();                                             // nobody leaves while its sums are read
  }
  tmem_fence_before_sync();
  __syncthreads();
  if (warp == 8 && lane == 0 && s.dead) {
    // What was requested still lands in this block's memory, whichever wait ran out.  Where no barrier of this block tells (a pair's
    // second block; a stage whose tokens were never asked for), the limit of a wait outlasts it: `drained` has no second phase.
    if (PAIR || ahead > issued) {
      mbar_wait(smem_addr(&s.drained), 0);
      mbar_wait(smem_addr(&s.drained), 1);
    }
    for (int i = 0; !PAIR && i < a.stages && i < issued; ++i) {
      if (--copy_stage < 0) copy_stage = a.stages - 1, copy_phase ^= 1;
      mbar_wait(smem_addr(&s.full[copy_stage]), copy_phase);
    }
  }
  __syncwarp();
  if constexpr (PAIR) cluster_sync();                           // neither block's memory or barriers are used by the other any more
  if (warp == 9) tmem_free<PAIR>(tmem, columns);
}

// ------------------------------------------------------------------ host
// The cut: tokens of a tile, blocks that share a reduction, pairs or single blocks, by what they are expected to take (us): a
// stage's bytes at what an SM gets from the L2 or its matrix instructions, the epilogue, and what a wave spends besides.  The
// constants are fitted to times of all cuts for 16 to 16384 tokens, 500 to 16384 channels and reductions over 1000 to 8192, e.g.
// 200 x 4096 x 4096: 208 tokens shared by four 12.4, by two 15.5, 64 tokens alone 14.2; 512 x 4096 x 4096: 128 tokens alone 15.1,
// 256 shared by two 17.2; pairs or single blocks, 16384 x 4096 x 8192 360 / 390, 16384 x 1024 x 1024 23.0 / 21.5.
void plan(MmArgs& a) {
  constexpr double kBytes = 100e3, kColumns = 950.;            // a microsecond: bytes of an SM, columns of a stage
  const int sms = device_info().sm_count;
  const int64_t least = (a.T + 255) / 256;
  const bool boxes = a.boxes;
  a.k_blocks = (a.K + kMmStageK - 1) / kMmStageK;
  double best = -1.;
  auto offer = [&](int tokens, int splits, bool pair) {
    const int step = boxes || pair ? 32 : 16;
    tokens = splits > 1 ? (tokens + 15) / 16 * 16 : (tokens + step - 1) / step * step;
    if (tokens > 256) return;
    const int channels = pair ? 2 * kMmChannels : kMmChannels;
    const int64_t channel_tiles = (a.N + channels - 1) / channels, tiles = channel_tiles * ((a.T + tokens - 1) / tokens);
    const int64_t blocks = tiles * splits * (pair ? 2 : 1), waves = (blocks + sms - 1) / sms;
    if (splits > 1 && blocks > sms) return;
    const double load = (kMmChannels + (pair ? tokens / 2 : tokens)) * kMmStageK / kBytes, multiply = tokens / kColumns;
    const double stages = (a.k_blocks + splits - 1) / splits * (load > multiply ? load : multiply);
    const double time = (double)waves * (stages + (splits > 1 ? 1.7 + tokens * 0.0075 : tokens * 0.006) + (pair ? 2. : 0.5));
    if (best >= 0. && time >= best) return;
    best = time;
    a.tokens = tokens;
    a.splits = splits;
    a.pair = pair;
    a.channel_tiles = (int)channel_tiles;
    a.tiles = (int)tiles;
  };
  for (const int64_t more : {1, 2, 3, 4, 6, 8}) {
    const int tokens = (int)((a.T + least * more - 1) / (least * more));
    if (more > 1 && tokens < 16) break;
    for (int splits = 1; splits <= kMmSplitsMost && a.k_blocks >= 2 * splits; splits *= 2) offer(tokens, splits, false);
    if (a.k_blocks < 2) offer(tokens, 1, false);
    if (tokens > 64) offer(tokens, 1, true);
  }
  a.boxes = boxes && a.splits == 1;
  a.columns = 32;
  while (a.columns < a.tokens) a.columns *= 2;
  a.stages = (kMmSmem - 1024 - (a.boxes ? kMmStaging : 0)) / ((kMmChannels + (a.pair ? a.tokens / 2 : a.tokens)) * kMmStageK);
  if (a.stages > kMmStagesMost) a.stages = kMmStagesMost;
}

template <typename T, bool SPLIT, bool PAIR> int launch(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& y, const MmArgs& a, cudaStream_t stream) {
  auto* kernel = int8_matmul_kernel<T, SPLIT, PAIR>;
  static std::atomic<uint64_t> raised{0};                       // devices whose limit of dynamic shared memory is raised
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (!(raised.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMmSmem) != cudaSuccess) return check_launch(), ACTNN_ERR_LAUNCH;
    raised.fetch_or(bit, std::memory_order_release);
  }
  const int sms = device_info().sm_count;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(SPLIT ? a.tiles * a.splits : PAIR ? 2 * (a.tiles < sms / 2 ? a.tiles : sms / 2) : a.tiles < sms ? a.tiles : sms);
  cfg.blockDim = dim3(kMmThreads);
  cfg.dynamicSmemBytes = kMmSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = SPLIT ? a.splits : PAIR ? 2 : 1;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.early ? 2 : 1;
  unsigned* gave_up = bulk_wait_counter();
  if (cudaLaunchKernelEx(&cfg, kernel, w, x, y, a, gave_up) != cudaSuccess) {
    cudaGetLastError();
    return ACTNN_ERR_LAUNCH;
  }
  return check_launch();
}
template <typename T> int launch_typed(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& y, const MmArgs& a, cudaStream_t stream) {
  return a.pair ? launch<T, false, true>(w, x, y, a, stream) : a.splits > 1 ? launch<T, true, false>(w, x, y, a, stream) : launch<T, false, false>(w, x, y, a, stream);
}

}  // namespace
}  // namespace actnn

using namespace actnn;

int actnn::int8_matmul_impl(const int8_t* tokens, const float* token_scale, const int8_t* weights, const float* channel_scale,
                            const void* bias, void* out, int64_t T, int64_t N, int64_t K, int64_t ld_tokens, int64_t ld_weights,
                            int dtype, bool early, actnn_stream_t stream) {
  if (T < 0 || N < 0 || K < 1 || K > 131072 || T > 0x7fffff00 || N > 0x7fffff00 || ld_tokens < K || ld_weights < K ||
      ld_tokens > ((int64_t)1 << 39) || ld_weights > ((int64_t)1 << 39)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (T == 0 || N == 0) return ACTNN_OK;
  if (!tokens || !token_scale || !weights || !channel_scale || !out) return ACTNN_ERR_NULL;
  if (!aligned(tokens, 16) || !aligned(weights, 16) || ld_tokens % 16 != 0 || ld_weights % 16 != 0) return ACTNN_ERR_ALIGN;
  const int size = dtype_size(dtype);
  if (!aligned(token_scale, 4) || !aligned(channel_scale, 4) || !aligned(bias, size) || !aligned(out, size)) return ACTNN_ERR_ALIGN;
  MmArgs a{};
  a.token_scale = token_scale; a.channel_scale = channel_scale; a.bias = bias; a.out = out;
  a.T = T; a.N = N; a.K = (int)K;
  a.vectors = N % 4 == 0 && aligned(out, 4 * size < 16 ? 4 * size : 16);
  a.early = early;
  a.boxes = N * size % 16 == 0 && aligned(out, 16);
  if ((N + kMmChannels - 1) / kMmChannels * ((T + 15) / 16) > 0x7fffffff) return ACTNN_ERR_SHAPE;
  plan(a);
  CUtensorMap w, x, y{};
  if (a.boxes && !map_values(&y, out, N, T, dtype, kMmChannels, kMmStaging / 4 / (kMmChannels * size))) return ACTNN_ERR_LAUNCH;
  if (!map_bytes(&w, weights, K, N, ld_weights, kMmStageK, kMmChannels, true) ||
      !map_bytes(&x, tokens, K, T, ld_tokens, kMmStageK, a.pair ? a.tokens / 2 : a.tokens, true)) return ACTNN_ERR_LAUNCH;
  switch (dtype) {
    case ACTNN_F32: return launch_typed<float>(w, x, y, a, (cudaStream_t)stream);
    case ACTNN_F16: return launch_typed<__half>(w, x, y, a, (cudaStream_t)stream);
    default: return launch_typed<__nv_bfloat16>(w, x, y, a, (cudaStream_t)stream);
  }
}

extern "C" int actnn_int8_matmul(const int8_t* tokens, const float* token_scale, const int8_t* weights, const float* channel_scale,
                                 const void* bias, void* out, int64_t T, int64_t N, int64_t K, int64_t ld_tokens,
                                 int64_t ld_weights, int dtype, actnn_stream_t stream) {
  return int8_matmul_impl(tokens, token_scale, weights, channel_scale, bias, out, T, N, K, ld_tokens, ld_weights, dtype, false, stream);
}
