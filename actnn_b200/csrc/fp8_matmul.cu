// Matrix product in 8-bit floating point with power-of-two scales for blocks of 128 along the reduction:
//
//   out[t, n] = sum_k x[t, k] * 2^ex[t, k / 128] * w[n, k] * 2^ew[n, k / 128] + bias[n]
//
// The matrix instructions apply the scales themselves (one for 32 values; a block's is named four times) and sum in fp32, so no partial
// sum leaves tensor memory before the end.  A layer's three products are this one: the gradient of the input reduces over output
// channels, that of the weight over tokens, each on operands coded along its reduction (fp8_codes.cu).
//
// The pipeline is that of the integer product (int8_matmul.cu): tiles of 128 channels (a lane of tensor memory each) by up to 224 tokens,
// one thread for the copies, one for the matrix instructions, eight warps that write one accumulator while the next one fills; the
// reduction split over a cluster where the tiles are too few; pairs of blocks on 256 channels where they are many.  Scales lie in global
// memory as the instructions read them, 512 bytes for 128 rows and four blocks: they come with the first stage of the four,
// go to tensor memory by tcgen05.cp, and each of the next stages names its byte of a column.  Two accumulators of 224 columns leave
// 64 for scales, four sets of 12; a wide one of 448 as many, three of 20: none is overwritten while instructions that read it may be under way.  Split sums
// are joined in the order of the blocks, so a shape's results are reproducible.
//
// 16384 x 4096 x 8192: 407 us in short runs, 2.7 PFLOP/s, 476 in long ones, where the power cap sets the clock; 8192 x 2048 x 4096 and its two
// gradients 60 to 64 each (2.2), in long runs 68 to 73;
// 200 x 4096 x 4096: 14, bound by what an SM gets from the L2 (51 bytes a cycle, 24 KB a stage) and latency (the weight's bytes from HBM 2.6).
//
// Every wait is bounded, with the integer product's rules: a block whose wait runs out writes nothing more, is counted, lets its copies
// and instructions end and leaves; the epilogue's warps leave together; of blocks that share a reduction none writes.
#include <algorithm>
#include <atomic>

#include "fp8.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace actnn {
namespace {

constexpr int kFpThreads = 320;                 // 8 epilogue warps, one for the copies, one for the matrix instructions
constexpr int kFpEpilogue = 256;
constexpr int kFpStagesMost = 8, kFpSplitsMost = 8;
constexpr int kFpStageK = 128;                  // bytes of the reduction in a stage
constexpr int kFpChannels = 128;
constexpr int kFpStaging = 32 * 1024;           // outputs on their way: two buffers for each half of the epilogue's warps
constexpr int kFpSmem = 216 * 1024;             // of the SM's 227 KB: stages with their scales, and 1 KB to align them
constexpr int kFpTokens = 224;                  // of an accumulator that has a twin
constexpr int kFpWide = 448;                    // of one that has none
constexpr int kFpScaleSets = 4;                 // at most, of columns of tensor memory

struct FpArgs {
  const void* bias;
  void* out;
  int64_t T, N;
  int K, tokens, stages, k_blocks, splits;      // tokens: columns of a tile
  int channel_tiles, tiles, columns;            // columns: of tensor memory, all
  int atoms, scale_rows_w, scale_rows_x;        // sets of 128 rows that a tile's tokens lie in; that the operands have
  int stage_scales, sets, set_columns;          // bytes of a stage's scales; sets of columns for them
  int first;                                    // of a wide tile: the tokens of its first half
  bool pair;                                    // tiles of 256 channels by pairs of blocks
  bool wide;                                    // one accumulator of two halves
  bool boxes;                                   // outputs leave as boxes of 128 channels
  bool vectors;                                 // four outputs of a token at a time are aligned
  bool early;                                   // the launch before this one makes the tokens' codes, and is not waited for sooner than they are read
};

struct FpShared {
  uint64_t full[kFpStagesMost], empty[kFpStagesMost], sum_full[2], sum_empty[2], drained;
  uint32_t tmem;
  int dead, gone;                               // a wait of the block has run out; of one of the blocks that share a reduction
};

// Tokens of a box: 8 KB of 128 channels.
template <typename T> constexpr int box_tokens() { return kFpStaging / 4 / (kFpChannels * (int)sizeof(T)); }
ACTNN_DEV void store_shared(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" :: "r"(at), "f"(v) : "memory"); }
ACTNN_DEV void store_shared(uint32_t at, __half v) { asm volatile("st.shared.u16 [%0], %1;" :: "r"(at), "h"(__half_as_ushort(v)) : "memory"); }
ACTNN_DEV void store_shared(uint32_t at, __nv_bfloat16 v) {
  asm volatile("st.shared.u16 [%0], %1;" :: "r"(at), "h"(__bfloat16_as_ushort(v)) : "memory");
}

// Waits for a phase; false once this or another wait of the block has run out.
ACTNN_DEV bool fp_wait(uint32_t bar, uint32_t parity, FpShared& s, unsigned* gave_up) {
  volatile int* dead = &s.dead;
  for (uint32_t i = 0; i < kBulkWaitTries; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*dead) return false;
  }
  *dead = 1;
  if (gave_up) atomicAdd(gave_up, 1u);
  return false;
}

// Whether a phase is complete: asked for the next stage before this one's work is issued, so that the answer's latency passes beside it.
ACTNN_DEV bool fp_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}

// Of a warp that issues by an elected lane: all of its lanes go on, or none.  A lane that left alone, because its own last try came a
// moment before the phase, would be missing where the others elect one.
ACTNN_DEV bool fp_warp_waits(bool ready, uint32_t bar, uint32_t parity, FpShared& s, unsigned* gave_up) {
  return __all_sync(kFull, ready || fp_wait(bar, parity, s, gave_up));
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
// WIDE (of a pair): one accumulator of up to 448 columns instead of two, since what an SM gets from the L2 limits the tiles of
// 192.  Its columns are two halves: while the epilogue has the second one, the matrix instructions begin the next tile with the first,
// for as many stages as there are, and then catch up.
template <typename T, bool SPLIT, bool PAIR, bool WIDE>
__global__ void __launch_bounds__(kFpThreads, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap tokens,
                  const __grid_constant__ CUtensorMap more_tokens, const __grid_constant__ CUtensorMap weight_scales, const __grid_constant__ CUtensorMap token_scales,
                  const __grid_constant__ CUtensorMap outputs, const FpArgs a, unsigned* gave_up) {
  extern __shared__ uint8_t dynamic_s[];
  __shared__ FpShared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stage0 = (smem_addr(dynamic_s) + 1023u) & ~1023u;
  const uint32_t rank = SPLIT || PAIR ? cluster_rank() : 0, split = SPLIT ? rank : 0;
  const int load_tokens = PAIR ? a.tokens / 2 : a.tokens, tile_channels = PAIR ? 2 * kFpChannels : kFpChannels;
  const uint32_t a_bytes = kFpChannels * kFpStageK, stage_bytes = a_bytes + load_tokens * kFpStageK, scale_bytes = 512 * (1 + a.atoms);
  const uint32_t scales0 = stage0 + a.stages * stage_bytes + (a.boxes ? kFpStaging : 0);
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
      mbar_init(smem_addr(&s.sum_empty[i]), (PAIR ? 2 : 1) * kFpEpilogue / 32);
    }
    mbar_init(smem_addr(&s.drained), 1);
    s.dead = s.gone = 0;
    mbar_init_fence();
  }
  const uint32_t columns = a.columns;
  if (warp == 9) tmem_alloc<PAIR>(smem_addr(&s.tmem), columns);
  tmem_fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();                           // both blocks have their barriers and their tensor memory
  if constexpr (SPLIT) cluster_arrive();                        // this block's flags are set
  tmem_fence_after_sync();
  const uint32_t tmem = s.tmem;

  // The copies' and the matrix instructions' warps go through their loops with all lanes, of which the first one issues: what a loop
  // counts is then uniform, and its addresses are where the instructions want them.  (A loop of one lane alone took 650 cycles a
  // stage, whatever it issued, 0.39 us where the matrix instructions of 192 tokens take 0.22.)
  const bool issues = lane == 0;
  int copy_stage = 0, issued = 0, ahead = 0;                    // of the copies, to the end
  uint32_t copy_phase = 0;
  bool copied = true;
  if (warp == 8) {                                              // ---------------- copies
    const int channel_step = (int)rank * kFpChannels * PAIR, token_step = (int)rank * load_tokens * PAIR;
    // Requests a box of a stage; of a pair, the first block's barrier counts.
    auto request = [&](uint32_t bar, uint32_t dst, const CUtensorMap* map, int x, int row) {
      if constexpr (PAIR) tile_load_pair(dst, map, x, row, peer_addr(bar, 0));
      else tile_load(dst, map, x, row, bar);
    };
    // The scales of four blocks come with the first of them that is multiplied.
    auto expect = [&](uint32_t bar, bool begins) {
      const uint32_t bytes = stage_bytes + (begins ? scale_bytes : 0);
      if (!PAIR || rank == 0) mbar_expect_tx(bar, PAIR ? 2 * bytes : bytes);
    };
    auto request_weights = [&](uint32_t bar, int stage, int k, bool begins, int row) {
      request(bar, stage0 + stage * stage_bytes, &weights, k * kFpStageK, row);
      if (begins) request(bar, scales0 + stage * a.stage_scales, &weight_scales, 0, 2 * ((k >> 2) * a.scale_rows_w + (row >> 7)));
    };
    if (a.early) {                                              // weights of the first stages before the tokens are there
      const int row = first_tile % a.channel_tiles * tile_channels + channel_step;
      for (ahead = 0; first_tile < a.tiles && ahead < a.stages && ahead < k_end - k_first; ++ahead) {
        const int k = k_first + ahead;
        const bool begins = ahead == 0 || (k & 3) == 0;
        const uint32_t bar = smem_addr(&s.full[ahead]);
        if (elect_one()) {
          expect(bar, begins);
          request_weights(bar, ahead, k, begins, row);
        }
      }
      grid_wait();
    }
    bool free = false;
    for (int tile = first_tile; copied && tile < a.tiles; tile += tile_step) {
      const int tt = tile / a.channel_tiles, row = (tile - tt * a.channel_tiles) * tile_channels + channel_step, t0 = tt * a.tokens;
      for (int k = k_first; k < k_end; ++k) {
        if (!(copied = fp_warp_waits(free, smem_addr(&s.empty[copy_stage]), copy_phase ^ 1, s, issues ? gave_up : nullptr))) break;
        const int now = copy_stage;
        if (++copy_stage == a.stages) copy_stage = 0, copy_phase ^= 1;
        free = fp_test(smem_addr(&s.empty[copy_stage]), copy_phase ^ 1);
        const bool begins = k == k_first || (k & 3) == 0;
        const uint32_t bar = smem_addr(&s.full[now]);
        if (elect_one()) {
          if (issued >= ahead) {
            expect(bar, begins);
            request_weights(bar, now, k, begins, row);
          }
          if constexpr (WIDE) {                                 // half of each half
            request(bar, stage0 + now * stage_bytes + a_bytes, &tokens, k * kFpStageK, t0 + (int)rank * (a.first / 2));
            request(bar, stage0 + now * stage_bytes + a_bytes + a.first / 2 * kFpStageK, &more_tokens, k * kFpStageK,
                    t0 + a.first + (int)rank * ((a.tokens - a.first) / 2));
          } else {
            request(bar, stage0 + now * stage_bytes + a_bytes, &tokens, k * kFpStageK, t0 + token_step);
          }
          if (begins) request(bar, scales0 + now * a.stage_scales + 512, &token_scales, 0, 2 * ((k >> 2) * a.scale_rows_x + (t0 >> 7)));
        }
        ++issued;
      }
    }
    // A pair's second block is there until what the first one's matrix instructions arrive at has been arrived at: the stages' barriers
    // and the one for the end.  (In their own block the warp that issues them waits for the end.)
    for (int i = 0, at = copy_stage; PAIR && copied && i < a.stages; ++i) {
      copied = fp_warp_waits(false, smem_addr(&s.empty[at]), copy_phase ^ (at < copy_stage ? 0 : 1), s, issues ? gave_up : nullptr);
      if (++at == a.stages) at = 0;
    }
    if (PAIR && copied) copied = fp_warp_waits(false, smem_addr(&s.drained), 0, s, issues ? gave_up : nullptr);
    __syncwarp();
  } else if (warp == 9) {                                       // ---------------- matrix instructions
    if (a.early) grid_wait();                                   // the limit of a wait is for copies, not for the launch before
    if (!PAIR || rank == 0) {
      const int first = WIDE ? a.first : a.tokens;
      const uint32_t instruction = fp8_instruction(tile_channels, first, 0), second = fp8_instruction(tile_channels, a.tokens - first, 0);
      const uint32_t one_byte = fp8_instruction(tile_channels, first, 1) - instruction, sets = tmem + (SPLIT || WIDE ? 1 : 2) * a.tokens;
      int stage = 0, buf = 0, set = 0;
      uint32_t phase = 0, buf_phase = 0, d = tmem, at_w = 0, shift = 0;
      bool ok = true;
      auto next = [&](int& at, uint32_t& at_phase) { if (++at == a.stages) at = 0, at_phase ^= 1; };
      // One lane: the scales of a stage that begins a set; the products of a stage, `half` of a wide tile.
      auto scales = [&](int at) {
        const uint32_t from = scales0 + at * a.stage_scales;
        scales_to_tmem<PAIR>(at_w, from);
        scales_to_tmem<PAIR>(at_w + 4, from + 512);
        if (a.atoms > 1) scales_to_tmem<PAIR>(at_w + 8, from + 1024);
        if (WIDE && a.atoms > 2) scales_to_tmem<PAIR>(at_w + 12, from + 1536);
        if (WIDE && a.atoms > 3) scales_to_tmem<PAIR>(at_w + 16, from + 2048);
      };
      auto multiply = [&](int at, int k, int half) {
        const uint32_t from = stage0 + at * stage_bytes;
        const uint64_t da = rows128_descriptor(from), db = rows128_descriptor(from + a_bytes + (half ? first / 2 * kFpStageK : 0));
        const uint32_t instr = (half ? second : instruction) + (k & 3) * one_byte, to = d + (half ? first : 0);
        const uint32_t at_x = at_w + 4 + shift + (half ? first / 32 : 0);
#pragma unroll
        for (int i = 0; i < kFpStageK / 32; ++i)                // 32 bytes further along the rows: 2 in units of 16 bytes
          mma_fp8<PAIR>(to, da + 2 * i, db + 2 * i, instr, at_w, at_x, k > k_first || i > 0);
      };
      for (int tile = first_tile; ok && tile < a.tiles; tile += tile_step) {
        if (!(ok = fp_warp_waits(false, smem_addr(&s.sum_empty[WIDE ? 0 : buf]), buf_phase ^ 1, s, issues ? gave_up : nullptr))) break;
        tmem_fence_after_sync();
        d = tmem + (WIDE ? 0 : buf * a.tokens);
        shift = (tile / a.channel_tiles * a.tokens & 127) / 32;                     // columns from a set of 128 tokens
        int k = k_first;
        if constexpr (WIDE) {                                   // a set of scales covers the stages that are caught up on
          const int head = min(min(a.stages, 4), k_end - k_first);
          int at = stage;
          uint32_t at_phase = phase;
          at_w = sets + set * a.set_columns;
          if (++set == a.sets) set = 0;
          for (int i = 0; ok && i < head; ++i) {
            if (!(ok = fp_warp_waits(false, smem_addr(&s.full[at]), at_phase, s, issues ? gave_up : nullptr))) break;
            if (elect_one()) {
              if (i == 0) scales(at);
              multiply(at, k_first + i, 0);
            }
            next(at, at_phase);
          }
          if (!ok || !(ok = fp_warp_waits(false, smem_addr(&s.sum_empty[1]), buf_phase ^ 1, s, issues ? gave_up : nullptr))) break;
          tmem_fence_after_sync();
          for (; k < k_first + head; ++k) {
            if (elect_one()) {
              multiply(stage, k, 1);
              mma_commit<PAIR>(smem_addr(&s.empty[stage]));
            }
            next(stage, phase);
          }
        }
        bool ready = false;
        for (; k < k_end; ++k) {
          if (!(ok = fp_warp_waits(ready, smem_addr(&s.full[stage]), phase, s, issues ? gave_up : nullptr))) break;
          const int now = stage;
          next(stage, phase);
          ready = fp_test(smem_addr(&s.full[stage]), phase);
          const bool begins = k == k_first || (k & 3) == 0;
          if (begins) {
            at_w = sets + set * a.set_columns;
            if (++set == a.sets) set = 0;
          }
          if (elect_one()) {
            if (begins) scales(now);
            multiply(now, k, 0);
            if constexpr (WIDE) multiply(now, k, 1);
            mma_commit<PAIR>(smem_addr(&s.empty[now]));
          }
        }
        if (!ok) break;
        if (elect_one()) mma_commit<PAIR>(smem_addr(&s.sum_full[WIDE ? 0 : buf]));
        if (WIDE || ++buf == 2) buf = 0, buf_phase ^= 1;
      }
      __syncwarp();
      if (elect_one()) {
        mma_commit<PAIR>(smem_addr(&s.drained));
        mbar_wait(smem_addr(&s.drained), 0);
      }
    }
    __syncwarp();
  } else {                                                      // ---------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    if (a.early) grid_wait();
    int buf = 0, box_buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = first_tile; tile < a.tiles; tile += tile_step) {
      const int tt = tile / a.channel_tiles, ct = tile - tt * a.channel_tiles;
      const int64_t t0 = (int64_t)tt * a.tokens, n = (int64_t)ct * tile_channels + rank * kFpChannels * PAIR + quarter * 32 + lane;
      const float b = n < a.N && a.bias ? to_float(reinterpret_cast<const T*>(a.bias)[n]) : 0.f;
      // One warp waits for the sums, the others for its word: sleepers wake up to a microsecond apart.
      const bool ok = warp != 0 || fp_wait(smem_addr(&s.sum_full[buf]), buf_phase, s, lane == 0 ? gave_up : nullptr);
      tmem_fence_after_sync();
      tmem_fence_before_sync();
      if (!epilogue_agrees(ok)) break;
      tmem_fence_after_sync();
      const uint32_t d = tmem + buf * a.tokens + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
      for (int part = 0; part < (WIDE ? 2 : 1); ++part) {
      const int begin = part ? a.first : 0, end = WIDE && !part ? a.first : a.tokens;
      if (!SPLIT && a.boxes) {
        // The warps of a half turn kBoxTokens columns into rows of 128 channels in shared memory, which one thread sends off as a
        // box while the next ones are made.
        constexpr int kBoxTokens = box_tokens<T>();
        for (int c = begin + half * kBoxTokens; c < end; c += 2 * kBoxTokens) {
          const uint32_t box = stage0 + a.stages * stage_bytes + (half * 2 + box_buf) * (kFpStaging / 4);
          if ((threadIdx.x & 127) == 0) tile_store_read<1>();                       // the buffer's last box has been read
          asm volatile("bar.sync %0, 128;" :: "r"(2 + half) : "memory");
#pragma unroll
          for (int k = 0; k < kBoxTokens; k += 16) {
            uint32_t r[16];
            tmem_load16(d + c + k, r);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              store_shared(box + ((k + i) * kFpChannels + quarter * 32 + lane) * sizeof(T), from_float<T>(__uint_as_float(r[i]) + b));
          }
          tile_store_fence();
          asm volatile("bar.sync %0, 128;" :: "r"(2 + half) : "memory");
          if ((threadIdx.x & 127) == 0) tile_store(&outputs, (int)(n - lane), (int)(t0 + c), box);
          box_buf ^= 1;
        }
      } else
      for (int c = begin + half * 16; c < end; c += 32) {
        uint32_t r[16];
        tmem_load16(d + c, r);
        tmem_load_wait();
        if constexpr (SPLIT) {                                  // [column][channel] over the stages, which are done with
          const uint32_t p = stage0 + c * (kFpChannels * 4) + (quarter * 32 + lane) * 4;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.u32 [%0], %1;" :: "r"(p + i * kFpChannels * 4), "r"(r[i]) : "memory");
        } else {
          T* o = reinterpret_cast<T*>(a.out) + (t0 + c) * a.N + n;
          const int left = (int)min((int64_t)16, a.T - t0 - c);
          if (n < a.N) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (i < left) o[i * a.N] = from_float<T>(__uint_as_float(r[i]) + b);
          }
        }
      }
      if constexpr (!SPLIT) {
        tmem_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) peer_arrive(peer_addr(smem_addr(&s.sum_empty[WIDE ? part : buf]), 0));
          else mbar_arrive(smem_addr(&s.sum_empty[buf]));
        }
      }
      }
      if (!SPLIT && (WIDE || ++buf == 2)) buf = 0, buf_phase ^= 1;
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
      const int64_t t0 = (int64_t)tt * a.tokens, n = (int64_t)ct * kFpChannels + lane * 4;
      float b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = n + i < a.N && a.bias ? to_float(reinterpret_cast<const T*>(a.bias)[n + i]) : 0.f;
      const int end = (int)min((int64_t)a.tokens, a.T - t0);
#pragma unroll 2
      for (int c = (int)split + a.splits * warp; c < end; c += 8 * a.splits) {
        float4 part[kFpSplitsMost];
#pragma unroll
        for (int k = 0; k < kFpSplitsMost; ++k)
          if (k < a.splits) part[k] = peer_load4(stage0 + c * (kFpChannels * 4) + lane * 16, k);
        float4 sum = part[0];
#pragma unroll
        for (int k = 1; k < kFpSplitsMost; ++k)
          if (k < a.splits) sum.x += part[k].x, sum.y += part[k].y, sum.z += part[k].z, sum.w += part[k].w;
        float2 out[2] = {make_float2(sum.x + b[0], sum.y + b[1]), make_float2(sum.z + b[2], sum.w + b[3])};
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
// The cut: tokens of a tile, blocks that share a reduction, pairs or single blocks, two accumulators or a wide one, by what they are
// expected to take (us): a stage, which is no shorter than its instructions take to issue, and what a tile takes besides.  Fitted to
// times of all cuts in long runs, where the power cap sets the clock; they are now: 16384 x 4096 x 8192, 448 tokens wide 476, 384 wide 479, 192 by
// pairs 493, by single blocks 564; 8192 x 2048 x 4096, 192 by pairs 73, 384 wide 76, 448 wide 80, 192 by single blocks 81; 4096 x 512 x 16384,
// 192 by single blocks 53, by pairs 64, 448 wide 68; 1024 x 4096 x 4096, 256 wide 20.5, 128 by pairs 25; 100 x 8192 x 2048, 64 shared by
// four 12.3, by two 16.4, alone 22.5.  Eight blocks that share a reduction find room for few such clusters at a time, and are offered where all do.
void plan(FpArgs& a) {
  const int sms = device_info().sm_count;
  const int64_t least = a.T <= kFpTokens ? 1 : (a.T + kFpTokens / 64 * 64 - 1) / (kFpTokens / 64 * 64);
  const bool boxes = a.boxes;
  a.k_blocks = (a.K + kFpStageK - 1) / kFpStageK;
  double best = -1.;
  auto offer = [&](int tokens, int splits, bool pair, bool wide) {
    // Scales of 32 tokens are a column, and the instructions want theirs to begin at an even one: where there are several tiles, they begin
    // at multiples of 64 tokens, and so does the second half of a wide one.
    const int step = wide ? 64 : a.T <= 16 && !boxes ? 16 : 32;
    tokens = (tokens + step - 1) / step * step;
    if (tokens < a.T) tokens = (tokens + 63) / 64 * 64;
    if (tokens > (wide ? kFpWide : kFpTokens) || (wide && tokens < 256)) return;
    const int channels = pair ? 2 * kFpChannels : kFpChannels;
    const int64_t channel_tiles = (a.N + channels - 1) / channels, tiles = channel_tiles * ((a.T + tokens - 1) / tokens);
    const int64_t blocks = tiles * splits * (pair ? 2 : 1), waves = (blocks + sms - 1) / sms;
    if (splits > 1 && blocks > (splits > 4 ? 64 : sms)) return;
    const double stage = wide ? tokens * 0.0017 : pair ? std::max(0.23, 0.15 + tokens * 0.00105) : std::max(splits > 1 ? 0.3 : 0.27, 0.2 + tokens * 0.0011);
    const double besides = wide ? 4.3 : pair ? 0.8 + tokens * 0.004 : splits > 1 ? 3. + tokens * 0.0135 : 0.4 + tokens * 0.004;
    const double time = (double)waves * ((a.k_blocks + splits - 1) / splits * stage + besides) + (pair ? 1. : 0.);
    if (best >= 0. && time >= best) return;
    best = time;
    a.tokens = tokens;
    a.splits = splits;
    a.pair = pair;
    a.wide = wide;
    a.channel_tiles = (int)channel_tiles;
    a.tiles = (int)tiles;
  };
  for (const int64_t more : {1, 2, 3, 4, 6, 8}) {
    const int tokens = (int)((a.T + least * more - 1) / (least * more));
    if (more > 1 && tokens < 16) break;
    for (int splits = 1; splits <= kFpSplitsMost && a.k_blocks >= 2 * splits; splits *= 2) offer(tokens, splits, false, false);
    if (a.k_blocks < 2) offer(tokens, 1, false, false);
    if (tokens > 64) offer(tokens, 1, true, false);
  }
  for (int tokens = 256; tokens <= kFpWide && tokens - 64 < a.T; tokens += 64) offer(tokens, 1, true, true);
  a.boxes = boxes && a.splits == 1;
  a.first = a.wide ? (a.tokens / 2 + 63) / 64 * 64 : a.tokens;
  int common = 128;
  while (a.tokens % common) common /= 2;
  a.atoms = (128 - common + a.tokens + 127) / 128;
  if (a.T <= a.tokens) a.atoms = (a.tokens + 127) / 128;
  a.set_columns = 4 + 4 * a.atoms;
  a.stage_scales = 512 * (1 + a.atoms);
  const int sums = (a.splits > 1 || a.wide ? 1 : 2) * a.tokens;
  a.sets = (512 - sums) / a.set_columns;
  if (a.sets > kFpScaleSets) a.sets = kFpScaleSets;
  a.columns = 32;
  while (a.columns < sums + a.sets * a.set_columns) a.columns *= 2;
  a.stages = (kFpSmem - 1024 - (a.boxes ? kFpStaging : 0)) / ((kFpChannels + (a.pair ? a.tokens / 2 : a.tokens)) * kFpStageK + a.stage_scales);
  if (a.stages > kFpStagesMost) a.stages = kFpStagesMost;
}

struct FpMaps { CUtensorMap w, x, x2, sw, sx, y; };
template <typename T, bool SPLIT, bool PAIR, bool WIDE> int launch(const FpMaps& m, const FpArgs& a, cudaStream_t stream) {
  auto* kernel = fp8_matmul_kernel<T, SPLIT, PAIR, WIDE>;
  static std::atomic<uint64_t> raised{0};                       // devices whose limit of dynamic shared memory is raised
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (!(raised.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFpSmem) != cudaSuccess) return check_launch(), ACTNN_ERR_LAUNCH;
    raised.fetch_or(bit, std::memory_order_release);
  }
  const int sms = device_info().sm_count;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(SPLIT ? a.tiles * a.splits : PAIR ? 2 * (a.tiles < sms / 2 ? a.tiles : sms / 2) : a.tiles < sms ? a.tiles : sms);
  cfg.blockDim = dim3(kFpThreads);
  cfg.dynamicSmemBytes = kFpSmem;
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
  if (cudaLaunchKernelEx(&cfg, kernel, m.w, m.x, m.x2, m.sw, m.sx, m.y, a, gave_up) != cudaSuccess) {
    cudaGetLastError();
    return ACTNN_ERR_LAUNCH;
  }
  return check_launch();
}
template <typename T> int launch_typed(const FpMaps& m, const FpArgs& a, cudaStream_t stream) {
  return a.wide        ? launch<T, false, true, true>(m, a, stream)
         : a.pair      ? launch<T, false, true, false>(m, a, stream)
         : a.splits > 1 ? launch<T, true, false, false>(m, a, stream)
                       : launch<T, false, false, false>(m, a, stream);
}

}  // namespace
}  // namespace actnn

using namespace actnn;

int actnn::fp8_matmul_impl(const uint8_t* tokens, const uint8_t* token_scales, const uint8_t* weights, const uint8_t* weight_scales,
                           const void* bias, void* out, int64_t T, int64_t N, int64_t K, int64_t ld_tokens, int64_t ld_weights,
                           int dtype, bool early, actnn_stream_t stream) {
  if (T < 0 || N < 0 || K < 1 || K > 0x7fffff00 || T > 0x7fffff00 || N > 0x7fffff00 || ld_tokens < K || ld_weights < K ||
      ld_tokens > ((int64_t)1 << 39) || ld_weights > ((int64_t)1 << 39)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (T == 0 || N == 0) return ACTNN_OK;
  if (!tokens || !token_scales || !weights || !weight_scales || !out) return ACTNN_ERR_NULL;
  if (!aligned(tokens, 16) || !aligned(weights, 16) || ld_tokens % 16 != 0 || ld_weights % 16 != 0) return ACTNN_ERR_ALIGN;
  const int size = dtype_size(dtype);
  if (!aligned(token_scales, 16) || !aligned(weight_scales, 16) || !aligned(bias, size) || !aligned(out, size)) return ACTNN_ERR_ALIGN;
  FpArgs a{};
  a.bias = bias; a.out = out;
  a.T = T; a.N = N; a.K = (int)K;
  a.vectors = N % 4 == 0 && aligned(out, 4 * size < 16 ? 4 * size : 16);
  a.early = early;
  a.boxes = N * size % 16 == 0 && aligned(out, 16);
  const int64_t rows_w = (N + 127) / 128, rows_x = (T + 127) / 128, groups = (K + 511) / 512;
  if ((N + kFpChannels - 1) / kFpChannels * ((T + 15) / 16) > 0x7fffffff || 2 * rows_w * groups > 0x7fffffff ||
      2 * rows_x * groups > 0x7fffffff) return ACTNN_ERR_SHAPE;
  plan(a);
  a.scale_rows_w = (int)rows_w;
  a.scale_rows_x = (int)rows_x;
  FpMaps m{};
  if (a.boxes && !map_values(&m.y, out, N, T, dtype, kFpChannels, kFpStaging / 4 / (kFpChannels * size))) return ACTNN_ERR_LAUNCH;
  if (!map_bytes(&m.w, weights, K, N, ld_weights, kFpStageK, kFpChannels, true) ||
      !map_bytes(&m.x, tokens, K, T, ld_tokens, kFpStageK, a.wide ? a.first / 2 : a.pair ? a.tokens / 2 : a.tokens, true) ||
      (a.wide && !map_bytes(&m.x2, tokens, K, T, ld_tokens, kFpStageK, (a.tokens - a.first) / 2, true)) ||
      !map_bytes(&m.sw, weight_scales, 256, 2 * rows_w * groups, 256, 256, 2, false) ||
      !map_bytes(&m.sx, token_scales, 256, 2 * rows_x * groups, 256, 256, 2 * a.atoms, false)) return ACTNN_ERR_LAUNCH;
  switch (dtype) {
    case ACTNN_F32: return launch_typed<float>(m, a, (cudaStream_t)stream);
    case ACTNN_F16: return launch_typed<__half>(m, a, (cudaStream_t)stream);
    default: return launch_typed<__nv_bfloat16>(m, a, (cudaStream_t)stream);
  }
}

extern "C" int actnn_fp8_matmul(const uint8_t* tokens, const uint8_t* token_scales, const uint8_t* weights, const uint8_t* weight_scales,
                                const void* bias, void* out, int64_t T, int64_t N, int64_t K, int64_t ld_tokens, int64_t ld_weights,
                                int dtype, actnn_stream_t stream) {
  return fp8_matmul_impl(tokens, token_scales, weights, weight_scales, bias, out, T, N, K, ld_tokens, ld_weights, dtype, false, stream);
}
