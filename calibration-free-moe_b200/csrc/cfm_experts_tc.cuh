// The gate/up and the down product of the routed experts on the 5th-generation tensor cores (sm_100a).
//
// One CTA per SM walks work items: a pass (an expert and up to TOKENS of its pairs) and a tile of 128 weight
// rows, which are 64 channels' gate and up rows, or 128 outputs of the down weight.  The weights are the
// instruction's first operand (M = 128), the tokens its second (N), so a weight goes from HBM to the tensor
// cores once per pass whatever the number of tokens.  Warps have roles:
//
//   * one thread of warp 4 brings weights by TMA into a ring of 16-KB stages in shared memory, across the
//     borders of the items: the ring is what hides the latency of HBM;
//   * the warps from 6 on bring the tokens' columns of the same stages, rows gathered with cp.async;
//   * one thread of warp 5 issues the products, into one of two places in tensor memory;
//   * warps 0 to 3 turn the sums of the item before into results meanwhile.
//
// Gate and up rows lie in the two halves of M; their sums meet through shared memory.  The down weight is
// channel-major, so its tile lies along M in memory (an MN-major operand).  Activations come as two BF16 terms,
// whose products add up in the same place: 16 bits of an activation, so that what is rounded is the output.
// Bound by HBM where an expert has few tokens; the down kernel starts on its weights before the kernel before it has
// ended.  With a hundred tokens per expert (1000 tokens of 64 experts: 108 and 78 us) a stage passes in 0.5 us: shared memory
// takes 34 and 52 KB of copies and gives the products 34 and 69 KB, some 540 and 940 of its cycles, and fewer stages are
// on their way.  HBM is at 5 and 3.7 TB/s then, L2 at 0.42 and 0.32 of its peak.  Not kept: two tiles per item that share the tokens'
// stages (261 us of a call against 216: three stages of tokens ahead are too few), weights and tokens in rings of
// their own (six stages of one and three of the other: 259; four: 241).
// Included by cfm_experts.cu inside its namespace.
#pragma once

constexpr int kTensorRows = 128;     // of weights, M
constexpr int kTensorColumns = 64;   // k of a stage: rows of 128 bytes, swizzled by 16-byte pieces
constexpr int kUpTile = 64;          // channels of an item

template <int TOKENS, bool DOWN>
struct Tensor {
  // Threads that gather tokens.  64 tokens of the 128-expert layer in passes of 16: 198 us with 64 of them, 201 with
  // 128; 1000 tokens of 64 experts in passes of 128: 274 with 64, 237 with 128.
  static constexpr int kGatherThreads = TOKENS <= 32 ? 64 : 128;
  static constexpr int kGatherRows = kGatherThreads / 8;  // a row of a stage is eight pieces
  static constexpr int kThreads = 192 + kGatherThreads;
  static constexpr int kWeightBytes = kTensorRows * 128;
  static constexpr int kTermBytes = TOKENS * 128;
  static constexpr int kStage = kWeightBytes + kTermBytes * (DOWN ? 2 : 1);
  static constexpr int kExchange = DOWN ? 0 : 2 * 4 * 8 * 32 * 4;  // two blocks of four warps' eight columns
  static constexpr int kRoom = 227 * 1024 - 1024 - 1024 - kExchange;  // less alignment and barriers
  static constexpr int kStages = kRoom / kStage < 12 ? kRoom / kStage : 12;
  static constexpr int kPlace = TOKENS > 128 ? 256 : TOKENS;  // columns of tensor memory of one of two places
  static constexpr uint32_t kTensorMemory = 2 * kPlace < 32 ? 32 : 2 * kPlace;
  static constexpr size_t kShared = 1024 + static_cast<size_t>(kStages) * kStage + kExchange;
  static_assert((kTensorMemory & (kTensorMemory - 1)) == 0 && kTensorMemory <= 512, "a power of two");
};

namespace tensor {

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: 1024 bytes from eight rows to the next eight.
// MN-major: eight k of 64 rows are 1024 bytes, the next 64 rows 8192 further.
__device__ __forceinline__ uint64_t descriptor(uint32_t address, bool across) {
  uint64_t d = (address & 0x3ffffu) >> 4;
  d |= static_cast<uint64_t>(across ? 8192 >> 4 : 1) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;  // descriptor version of sm_100
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// FP32 sums of BF16 operands, M = 128; the first operand K-major or, `across`, MN-major.
__device__ __forceinline__ uint32_t instruction(int columns, bool across) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (across ? 1u << 15 : 0u) | (static_cast<uint32_t>(columns >> 3) << 17) |
         (static_cast<uint32_t>(kTensorRows >> 4) << 24);
}

__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t what, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"(accumulate)
      : "memory");
}

// A box of the tensor map from (x, y) on; x in elements, a multiple of 8.
__device__ __forceinline__ void copy_box(uint32_t shared, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(shared),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// Arrives at the barrier once the thread's cp.async copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// All of the four result warps, once all have come: whether every one of them is alive.
__device__ __forceinline__ bool result_warps_agree(int alive) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(alive)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void result_warps_meet() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

}  // namespace tensor

// grid: at most one CTA per SM.  `weights`: the map of the weight with boxes of 64 columns and 64 rows.
template <int TOKENS, bool DOWN>
__global__ void __launch_bounds__(Tensor<TOKENS, DOWN>::kThreads, 1)
    k_experts_tensor(Experts L, Scratch s, const __nv_bfloat16* hidden, const __grid_constant__ CUtensorMap weights) {
  using S = Tensor<TOKENS, DOWN>;
  using namespace tc;
  using namespace tensor;
  extern __shared__ uint8_t tensor_shared[];
  // Barriers: a stage's weights have landed, its tokens have, it may be filled again; per place in tensor
  // memory, its sums are complete, it may be written; the last products have ended after a wait that ran out.
  __shared__ uint64_t barriers[3 * S::kStages + 5];
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag, late_flag, s_filled;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(kFull, tid >> 5, 0);  // known to be the same in all lanes
  const uint32_t abort = shared_u32(&abort_flag), late = shared_u32(&late_flag);
  const uint32_t ring = (shared_u32(tensor_shared) + 1023u) & ~1023u;
  const uint32_t weights_in = shared_u32(barriers), tokens_in = weights_in + 8 * S::kStages, freed = tokens_in + 8 * S::kStages;
  const uint32_t summed = freed + 8 * S::kStages, taken = summed + 16, drained = taken + 16;
  if (warp == 5 && lane == 0) {
    abort_flag = late_flag = s_filled = 0;
    for (int i = 0; i < S::kStages; ++i) {
      barrier_init(weights_in + 8 * i, 1);
      barrier_init(tokens_in + 8 * i, S::kGatherThreads);
      barrier_init(freed + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      barrier_init(summed + 8 * i, 1);
      barrier_init(taken + 8 * i, 4);
    }
    barrier_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_u32(&tmem_holder)),
                 "n"(S::kTensorMemory)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_holder;

  // The passes are of the kernel before the down kernel's predecessor, which let this one be scheduled only
  // once it had seen them itself; so only what reads the predecessor's results waits for it.
  if (!DOWN) {
    grid_dependency_wait();
    grid_dependency_release();
  }
  const int I = L.I, H = L.H;
  const int tiles = DOWN ? H / kTensorRows : (I + kUpTile - 1) / kUpTile;
  const int chunks = DOWN ? (I + kTensorColumns - 1) / kTensorColumns : H / kTensorColumns;
  const int items = __ldcg(&s.counts[0]) * tiles;
  // Expert, first pair, pairs.  Each role asks for an item's pass while it is at the item before.
  auto pass_of = [&](int item) { return item < items ? __ldcg(&s.passes[item / tiles]) : make_int4(0, 0, 0, 0); };
  const int step = gridDim.x;

  if (warp == 4) {
    // ---- weights ----
    if (elect_lane()) {
      int alive = 1, filled = 0, stage = 0;
      uint32_t turn = 1;  // parity of the round before; the first round finds all stages free
      int4 next = pass_of(blockIdx.x);
      for (int item = blockIdx.x; item < items && alive; item += step) {
        const int e = next.x, tile = item % tiles;
        next = pass_of(item + step);
        for (int c = 0; c < chunks; ++c) {
          const uint32_t bar = weights_in + 8 * stage, to = ring + stage * S::kStage;
          if (filled >= S::kStages) {
            barrier_wait(freed + 8 * stage, turn, abort, alive);
            if (!alive) break;
          }
          barrier_expect(bar, S::kWeightBytes);
          if (DOWN) {
            const int x = tile * kTensorRows, y = e * I + c * kTensorColumns;
            copy_box(to, &weights, x, y, bar);
            copy_box(to + 8192, &weights, x + 64, y, bar);
          } else {
            const int x = c * kTensorColumns, y = e * 2 * I + tile * kUpTile;
            copy_box(to, &weights, x, y, bar);
            copy_box(to + 8192, &weights, x, y + I, bar);
          }
          ++filled;
          if (++stage == S::kStages) {
            stage = 0;
            turn ^= 1;
          }
        }
      }
      s_filled = filled;
    }
    __syncwarp();
  } else if (warp == 5) {
    // ---- products ----
    if (elect_lane()) {
      int alive = 1, stage = 0, round = 0;
      uint32_t turn = 0;
      int4 next = pass_of(blockIdx.x);
      for (int item = blockIdx.x; item < items && alive; item += step, ++round) {
        const int count = next.z, place = round & 1;
        next = pass_of(item + step);
        const uint32_t sums = tmem + place * S::kPlace, what = instruction((count + 15) / 16 * 16, DOWN);
        if (round >= 2) barrier_wait(taken + 8 * place, ((round >> 1) - 1) & 1, abort, alive);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int c = 0; c < chunks && alive; ++c) {
          barrier_wait(weights_in + 8 * stage, turn, abort, alive);
          barrier_wait(tokens_in + 8 * stage, turn, abort, alive);
          if (!alive) break;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tokens came by ordinary copies
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t from = ring + stage * S::kStage;
          const uint64_t a = descriptor(from, DOWN), b = descriptor(from + S::kWeightBytes, false);
          const int steps = DOWN ? min(4, (I - c * kTensorColumns) / 16) : 4;
          for (int k = 0; k < steps; ++k) {
            product(sums, a + k * (DOWN ? 2048 >> 4 : 32 >> 4), b + k * (32 >> 4), what, c + k > 0);
            if (DOWN) product(sums, a + k * (2048 >> 4), b + (S::kTermBytes >> 4) + k * (32 >> 4), what, 1);
          }
          mma_commit(freed + 8 * stage);
          if (++stage == S::kStages) {
            stage = 0;
            turn ^= 1;
          }
        }
        if (alive) mma_commit(summed + 8 * place);
      }
      if (!alive) {  // nothing may outlive the CTA
        mma_commit(drained);
        barrier_wait(drained, 0, late, alive, CFM_SCREEN_DRAIN_NS);
      }
    }
    __syncwarp();
  } else if (warp >= 6) {
    // ---- tokens ----
    if (DOWN) {
      grid_dependency_wait();
      grid_dependency_release();
    }
    const int at = tid - 192, row0 = at >> 3, piece = at & 7;
    const uint32_t place = row0 * 128 + ((piece ^ (row0 & 7)) << 4);
    constexpr int kRows = (TOKENS + S::kGatherRows - 1) / S::kGatherRows;
    const int32_t* list = DOWN ? s.pairs : s.tokens;
    int alive = 1, filled = 0, stage = 0;
    uint32_t turn = 1;
    // Rows are asked for an item ahead, passes two.
    int row[kRows], next_row[kRows];
    auto rows_of = [&](const int4& pass) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int t = row0 + S::kGatherRows * j;
        next_row[j] = t < pass.z ? __ldcg(&list[pass.y + t]) : -1;
      }
    };
    rows_of(pass_of(blockIdx.x));
    int4 next = pass_of(blockIdx.x + step);
    for (int item = blockIdx.x; item < items && alive; item += step) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) row[j] = next_row[j];
      rows_of(next);
      next = pass_of(item + 2 * step);
      for (int c = 0; c < chunks; ++c) {
        if (filled >= S::kStages) barrier_wait(freed + 8 * stage, turn, abort, alive);
        if (!__all_sync(kFull, alive)) {
          alive = 0;
          break;
        }
        const uint32_t to = ring + stage * S::kStage + S::kWeightBytes + place;
        const int column = c * kTensorColumns + 8 * piece;
        if (!DOWN || column < I) {
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            if (row[j] < 0) continue;
            if (DOWN) {
              const size_t from = static_cast<size_t>(row[j]) * I + column;
              copy_async16(to + j * S::kGatherRows * 128, s.activations + from);
              copy_async16(to + S::kTermBytes + j * S::kGatherRows * 128, s.rests + from);
            } else {
              copy_async16(to + j * S::kGatherRows * 128, hidden + static_cast<size_t>(row[j]) * H + column);
            }
          }
        }
        copies_arrive(tokens_in + 8 * stage);
        ++filled;
        if (++stage == S::kStages) {
          stage = 0;
          turn ^= 1;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- results ----
    if (DOWN) {
      grid_dependency_wait();
      grid_dependency_release();
    }
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    float* exchange = reinterpret_cast<float*>(tensor_shared + (ring - shared_u32(tensor_shared)) + S::kStages * S::kStage);
    int alive = 1, round = 0, turn = 0;
    int4 next = pass_of(blockIdx.x);
    for (int item = blockIdx.x; item < items; item += step, ++round) {
      const int4 pass = next;
      next = pass_of(item + step);
      const int count = pass.z, tile = item % tiles, place = round & 1;
      int pairs[(TOKENS + 31) / 32];
#pragma unroll
      for (int j = 0; j < (TOKENS + 31) / 32; ++j) pairs[j] = 32 * j + lane < count ? __ldcg(&s.pairs[pass.y + 32 * j + lane]) : 0;
      barrier_wait(summed + 8 * place, (round >> 1) & 1, abort, alive);
      if (!result_warps_agree(alive)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int block = 0; block < TOKENS / 16; ++block) {
        if (16 * block >= count) break;
        int bits[16];
        load_columns16(tmem + place * S::kPlace + lanes + 16 * block, bits);
        load_wait();
        if (DOWN) {
          const int h = tile * kTensorRows + 32 * warp + lane;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int pair = __shfl_sync(kFull, pairs[block / 2], (16 * block + i) & 31);
            if (16 * block + i < count) s.sums[static_cast<size_t>(pair) * H + h] = __int_as_float(bits[i]);
          }
        } else {
          // Gate rows are with warps 0 and 1, which finish the first eight columns, up rows with 2 and 3.
          const bool has_gate = warp < 2;
          float* mine = exchange + (turn * 4 + warp) * 256 + lane;
#pragma unroll
          for (int i = 0; i < 8; ++i) mine[32 * i] = __int_as_float(has_gate ? bits[8 + i] : bits[i]);
          result_warps_meet();
          const float* other = exchange + (turn * 4 + (warp ^ 2)) * 256 + lane;
          turn ^= 1;
          const int channel = tile * kUpTile + 32 * (warp & 1) + lane;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int token = 16 * block + (has_gate ? i : 8 + i);
            const float own = __int_as_float(has_gate ? bits[i] : bits[8 + i]), from = other[32 * i];
            const int pair = __shfl_sync(kFull, pairs[block / 2], token & 31);
            if (token < count && channel < I)
              store_activation(s, static_cast<size_t>(pair) * I + channel,
                               gated(has_gate ? own : from, has_gate ? from : own, L.activation));
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      barrier_arrive(taken + 8 * place, lane == 0);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 4) {
    if (abort_flag) {
      // Each stage's last weights.  (Where no wait ran out, the products have read all of them.)
      int alive = 1;
      const int filled = s_filled;
      for (int p = 0; p < min(filled, S::kStages); ++p)
        barrier_wait(weights_in + 8 * p, ((filled - p - 1) / S::kStages) & 1, late, alive, CFM_SCREEN_DRAIN_NS);
      __syncwarp();
      if (lane == 0) atomicExch(s.status, 1);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTensorMemory) : "memory");
  }
}
