// The routed experts of one MoE layer as a whole (sm_100a): for every token the router-weighted sum over its
// experts of D_e (phi(G_e x) * (U_e x)), all channels, from the weights as the sparse reader keeps them.
//
// A call is bound by the weights of the experts that some token is routed to, so the (token, slot) pairs are
// grouped by expert and each weight is read once for all tokens of its expert:
//   group   the list of pairs by expert, and the passes over the experts
//   up      gate and up rows, activation, two BF16 terms [pair, I]
//   down    channel-major down rows, FP32 [pair, H]
//   mix     router weights, sum over a token's slots in their order, BF16
// up and down are cfm_experts_tc.cuh's; calls of few pairs have two kernels of their own, without lists.
// Sums are FP32.  The tensor cores take the type of the weights, so an activation goes to them as two BF16
// terms, its value rounded and what that leaves: at most 2^-16 of it is lost, beside the 2^-8 of the output's rounding.
// (Rounded once to BF16 they would have added as much as that: 0.0024 of the output's norm instead of 0.0016.)
// A pair's numbers do not depend on its place in the list nor on the other pairs: a token's output does not depend
// on the tokens beside it, but for calls of few pairs, whose kernels add in another order.
#include "cfm_device.cuh"
#include "cfm_launch.cuh"
#include "cfm_tc.cuh"

#include "cfm_b200.h"

#include <cuda.h>

#include <algorithm>
#include <type_traits>

namespace cfm {
namespace {

constexpr int kMaxExperts = 4096;
constexpr int kLeastPass = 32;    // pairs that the smallest pass of the tensor-core path takes

struct Experts {
  int H, I, E, K, activation;
  const __nv_bfloat16* gate_up;  // [E, 2 I, H]
  const __nv_bfloat16* down;     // [E, I, H]
};

struct Scratch {
  int32_t* pairs;    // [C K] pairs by expert
  int32_t* tokens;   // [C K] their tokens
  int4* passes;      // expert, first pair, pairs: of the tensor-core path
  int32_t* counts;   // [4] number of passes
  int32_t* status;   // [4] device-side errors
  __nv_bfloat16* activations;  // [C K, I]
  __nv_bfloat16* rests;        // [C K, I] what the activations' rounding leaves
  float* sums;                 // [C K, H]
};

struct Routes {
  const void* ids;
  const void* weights;
  const uint8_t* padding;
  int tokens, ids64, weights16;

  // The expert of a pair, -1 where it has none.  (From L2: a kernel may ask before its predecessor has ended.)
  __device__ int expert(int pair, int K, int E) const {
    if (padding && __ldcg(&padding[pair / K])) return -1;
    const int64_t e = ids64 ? __ldcg(&static_cast<const long long*>(ids)[pair]) : __ldcg(&static_cast<const int32_t*>(ids)[pair]);
    return e >= 0 && e < E ? static_cast<int>(e) : -1;
  }
  __device__ float weight(int pair) const {
    return weights16 ? __bfloat162float(__ldcg(&static_cast<const __nv_bfloat16*>(weights)[pair]))
                     : __ldcg(&static_cast<const float*>(weights)[pair]);
  }
};

// phi(g) u in FP32.  SiLU: g / (1 + e^-g); GELU, tanh form: g / (1 + e^(-2 z)), z = sqrt(2 / pi) (g + 0.044715 g^3).
__device__ __forceinline__ float gated(float g, float u, int activation) {
  const float z = activation == CFM_ACT_GELU_TANH ? 1.59576912f * (g + 0.044715f * g * g * g) : g;
  return __fdividef(g, 1.0f + __expf(-z)) * u;
}

__device__ __forceinline__ void store_activation(const Scratch& s, size_t at, float a) {
  const __nv_bfloat16 rounded = __float2bfloat16_rn(a);
  const float value = __bfloat162float(rounded);
  s.activations[at] = rounded;
  s.rests[at] = __float2bfloat16_rn(fabsf(value) < __builtin_huge_valf() ? a - value : 0.0f);  // of inf and NaN nothing
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- group: one CTA --------------------------------------------------------------------------------
// All latency (9 us of a call of 64 tokens when every pair was looked at twice and three sums were scanned): a
// thread keeps its pairs' experts and their places among the expert's pairs, which one pass of atomics gives,
// and the two sums are scanned as one number.  The order of an expert's pairs is as it comes.  The list is put in order in shared
// memory: 8000 pairs stored one by one took this CTA 9 of its 16 us.
constexpr int kGroupThreads = 1024;
constexpr int kGroupKept = 8;  // pairs of a thread that stay in registers; of larger calls the rest is looked at twice
constexpr int64_t kMostPairs = 1 << 24;

// `tokens`: pairs of a pass.
__global__ void __launch_bounds__(kGroupThreads) k_group_pairs(Routes routes, int E, int K, int tokens, Scratch s) {
  extern __shared__ int group_shared[];
  __shared__ uint64_t warps[32];
  int* list = group_shared;                                    // [kGroupKept * kGroupThreads] pairs by expert
  int* count = group_shared + kGroupKept * kGroupThreads;     // [E], then the first place of every expert
  const int tid = threadIdx.x, lane = tid & 31, pairs = routes.tokens * K;
  for (int e = tid; e < E; e += kGroupThreads) count[e] = 0;
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_release();
  int expert[kGroupKept], rank[kGroupKept];
#pragma unroll
  for (int j = 0; j < kGroupKept; ++j) {
    const int p = tid + j * kGroupThreads;
    expert[j] = p < pairs ? routes.expert(p, K, E) : -1;
  }
#pragma unroll
  for (int j = 0; j < kGroupKept; ++j)
    if (expert[j] >= 0) rank[j] = atomicAdd(&count[expert[j]], 1);
  const bool fits = pairs <= kGroupKept * kGroupThreads;
  if (!fits) {
    __syncthreads();  // the places are among the pairs kept
    for (int p = tid + kGroupKept * kGroupThreads; p < pairs; p += kGroupThreads) {
      const int e = routes.expert(p, K, E);
      if (e >= 0) atomicAdd(&count[e], 1);
    }
  }
  __syncthreads();
  // Pairs and passes before those of this thread, in one number.
  constexpr int kPassBits = 24;
  const int per = (E + kGroupThreads - 1) / kGroupThreads, from = min(E, tid * per), to = min(E, from + per);
  uint64_t mine = 0;
  for (int e = from; e < to; ++e)
    if (const int n = count[e])
      mine += static_cast<uint64_t>(n) | static_cast<uint64_t>((n + tokens - 1) / tokens) << kPassBits;
  uint64_t sum = mine;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const uint64_t other = __shfl_up_sync(kFull, sum, w);
    if (lane >= w) sum += other;
  }
  if (lane == 31) warps[tid >> 5] = sum;
  __syncthreads();
  if (tid < 32) {
    uint64_t all = warps[tid];
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const uint64_t other = __shfl_up_sync(kFull, all, w);
      if (lane >= w) all += other;
    }
    warps[tid] = all;
  }
  __syncthreads();
  const uint64_t before = sum - mine + (tid >= 32 ? warps[(tid >> 5) - 1] : 0);
  int offset = static_cast<int>(before & ((1u << kPassBits) - 1)), part = static_cast<int>(before >> kPassBits);
  for (int e = from; e < to; ++e) {
    const int n = count[e];
    count[e] = offset;
    for (int at = 0; at < n; at += tokens) s.passes[part++] = make_int4(e, offset + at, min(tokens, n - at), 0);
    offset += n;
  }
  if (tid == 0) s.counts[0] = static_cast<int>(warps[31] >> kPassBits);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroupKept; ++j) {
    if (expert[j] < 0) continue;
    const int p = tid + j * kGroupThreads, at = count[expert[j]] + rank[j];
    if (fits) {
      list[at] = p;
    } else {
      s.pairs[at] = p;
      s.tokens[at] = p / K;
    }
  }
  if (fits) {
    __syncthreads();
    const int grouped = static_cast<int>(warps[31] & ((1u << kPassBits) - 1));
    for (int at = tid; at < grouped; at += kGroupThreads) {
      const int p = list[at];
      s.pairs[at] = p;
      s.tokens[at] = p / K;
    }
    return;
  }
  // The other pairs come behind those.
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroupKept; ++j)
    if (expert[j] >= 0) atomicAdd(&count[expert[j]], 1);
  __syncthreads();
  for (int p = tid + kGroupKept * kGroupThreads; p < pairs; p += kGroupThreads) {
    const int e = routes.expert(p, K, E);
    if (e < 0) continue;
    const int at = atomicAdd(&count[e], 1);
    s.pairs[at] = p;
    s.tokens[at] = p / K;
  }
}

// ---- few pairs -------------------------------------------------------------------------------------
// Calls of up to 16 pairs in two launches (two tokens of the 128-expert layer 35 us, 43 on the tensor-core path; three would take 50
// and 50, four 65 and 62).  The weights go from global memory straight into the registers of
// warp-level tensor-core products (m16n8k16), whose eight columns are the tokens of an expert.  Every warp
// groups the pairs by itself, a pair per lane.
constexpr int kFewPairs = 16;

struct Few {
  int e;          // expert, -1: there are fewer
  unsigned mask;  // its pairs
};
// Of a warp, a pair per lane.
struct FewGroups {
  int e;           // the lane's expert
  unsigned same;   // lanes with that expert
  unsigned first;  // the first lane of every busy expert

  __device__ FewGroups(const Routes& routes, int K, int E) {
    const int lane = threadIdx.x & 31;
    e = lane < routes.tokens * K ? routes.expert(lane, K, E) : -1;
    same = __match_any_sync(kFull, e);
    first = __ballot_sync(kFull, e >= 0 && lane == __ffs(same) - 1);
  }
  __device__ int experts() const { return __popc(first); }
  // The `which`-th busy expert, in the order of first pairs.
  __device__ Few group(int which) const {
    if (which >= experts()) return {-1, 0};
    unsigned rest = first;
    for (int i = 0; i < which; ++i) rest &= rest - 1;
    const int from = __ffs(rest) - 1;
    Few few;
    few.e = __shfl_sync(kFull, e, from);
    few.mask = __shfl_sync(kFull, same, from);
    return few;
  }
  // The place of the lane's expert among the busy ones, -1 where it has none.
  __device__ int which() const { return e < 0 ? -1 : __popc(first & ((1u << (__ffs(same) - 1)) - 1)); }
};
// The pair at a place among the set bits, -1 behind them.
__device__ __forceinline__ int pair_at(unsigned mask, int place) {
  for (int i = 0; i < place; ++i) mask &= mask - 1;
  return __ffs(mask) - 1;
}

__device__ __forceinline__ void prefetch_row(const void* row, int bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row), "r"(bytes) : "memory");
}

constexpr int kFewUpThreads = 128;
constexpr int kFewUpWarps = kFewUpThreads / 32;
constexpr int kFewUpAhead = 4;  // steps of 32 columns whose rows are on their way
constexpr int kFewUpPerSm = 6;
constexpr int kFewUpBlock = 64;  // columns

// Items are eight channels of an expert; a CTA's warps share the columns, and it asks for its next item's first
// rows before it adds up the sums of the last.  A thread has 16 bytes of a gate row and of an up row, whose elements
// are the k of two instructions, and the same of a token's row; gate and up of a channel end in one thread.
__global__ void __launch_bounds__(kFewUpThreads, kFewUpPerSm)
    k_few_up(Experts L, Scratch s, Routes routes, const __nv_bfloat16* hidden) {
  __shared__ float sums[kFewUpWarps][4][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  grid_dependency_release();
  // A warp's columns are every fourth block of kFewUpBlock.
  constexpr int kPer = kFewUpBlock / 32;
  const int steps = (L.H / kFewUpBlock - warp + kFewUpWarps - 1) / kFewUpWarps * kPer, at = kFewUpBlock * warp + 8 * t, tiles = L.I / 8;
  auto column = [](int step) { return step / kPer * (kFewUpWarps * kFewUpBlock) + step % kPer * 32; };
  const FewGroups groups(routes, L.K, L.E);
  Few few = {};
  int count = 0, c0 = 0, pass = 0, pair = -1;
  const __nv_bfloat16 *gate, *up, *x;
  uint4 a[kFewUpAhead], b[kFewUpAhead], v[kFewUpAhead];
  auto fetch = [&](int i, int step) {
    a[i] = load_stream16(gate + column(step));
    b[i] = load_stream16(up + column(step));
    v[i] = pair >= 0 ? __ldg(reinterpret_cast<const uint4*>(x + column(step))) : make_uint4(0, 0, 0, 0);
  };
  // The first rows of a pass over an item.
  auto start = [&](int from) {
    pass = from;
    pair = pair_at(few.mask, pass + g);
    x = hidden + static_cast<size_t>(max(pair, 0) / L.K) * L.H + at;
#pragma unroll
    for (int i = 0; i < kFewUpAhead; ++i)
      if (i < steps) fetch(i, i);
  };
  auto open = [&](int item) {
    few = groups.group(item / tiles);
    if (few.e < 0) return;
    count = __popc(few.mask);
    c0 = item % tiles * 8;
    gate = L.gate_up + (static_cast<size_t>(few.e) * 2 * L.I + c0 + g) * L.H + at;
    up = gate + static_cast<size_t>(L.I) * L.H;
    start(0);
  };
  int item = blockIdx.x;
  open(item);
  while (few.e >= 0) {
    float acc[4] = {};
    for (int from = 0; from < steps; from += kFewUpAhead) {
#pragma unroll
      for (int i = 0; i < kFewUpAhead; ++i) {
        if (from + i >= steps) break;
        mma_bf16(acc, a[i].x, b[i].x, a[i].y, b[i].y, v[i].x, v[i].y);
        mma_bf16(acc, a[i].z, b[i].z, a[i].w, b[i].w, v[i].z, v[i].w);
        if (from + i + kFewUpAhead < steps) fetch(i, from + i + kFewUpAhead);
      }
    }
    const unsigned mask = few.mask;
    const int tokens = min(8, count - pass), first = pass, channels = c0;
    // The down rows of these channels, one after another in memory, come to L2 while the sums are added up and the
    // next kernel starts.
    if (tid < 8 && pass == 0) prefetch_row(L.down + (static_cast<size_t>(few.e) * L.I + c0 + tid) * L.H, 2 * L.H);
    if (pass + 8 < count) {
      start(pass + 8);
    } else {
      item += gridDim.x;
      open(item);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][i][lane] = acc[i];
    __syncthreads();
    if (tid < 8 * tokens) {
      const int channel = tid & 7, token = tid >> 3, from = 4 * channel + (token >> 1);
      float gu[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * half + (token & 1);
        float sum = sums[0][i][from];
#pragma unroll
        for (int j = 1; j < kFewUpWarps; ++j) sum += sums[j][i][from];
        gu[half] = sum;
      }
      store_activation(s, static_cast<size_t>(pair_at(mask, first + token)) * L.I + channels + channel,
                       gated(gu[0], gu[1], L.activation));
    }
    __syncthreads();
  }
}

constexpr int kFewDownThreads = 256;
constexpr int kFewDownWarps = kFewDownThreads / 32;
constexpr int kFewDownColumns = 64;  // of a cluster
constexpr int kFewDownAhead = 4;     // steps of 16 channels whose rows are on their way
constexpr int kFewRanks = 8;         // CTAs of a cluster

// grid (8 H / 64): a cluster has 64 outputs of all pairs, its CTAs share the experts, of which each has SPLITS parts of the
// channels; a CTA's warps share a part.  A thread has 16 bytes, eight outputs, of four channels'
// rows; the first operand's registers pair two channels of one output, which two byte permutations per pair of
// words do.  The first rows are on their way before the kernel before this one has ended.
// A token's bits do not depend on the tokens beside it: a pair's warps and parts are added in their order, a token's pairs in
// that of its slots.  So the parts go by K, not by how many experts a call has.
template <int SPLITS>
__global__ void __launch_bounds__(kFewDownThreads, 2)
    k_few_down(Experts L, Scratch s, Routes routes, __nv_bfloat16* out) {
  __shared__ float parts[kFewDownWarps][8][kFewDownColumns];
  __shared__ float total[kFewPairs][kFewDownColumns];  // of a pair, the channels of this CTA
  __shared__ float weights[kFewPairs];
  __shared__ int units[kFewPairs];  // a pair's first unit, -1: it has no expert
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % kFewRanks, h0 = blockIdx.x / kFewRanks * kFewDownColumns;
  const FewGroups groups(routes, L.K, L.E);
  const int experts = groups.experts();
  const float weight = tid < kFewPairs && groups.e >= 0 ? routes.weight(tid) : 0.0f;
  if (tid < kFewPairs) units[tid] = groups.e >= 0 ? groups.which() * SPLITS : -1;
  bool waited = false;
  for (int unit = rank; unit < experts * SPLITS; unit += kFewRanks) {
    const Few few = groups.group(unit / SPLITS);
    const int count = __popc(few.mask), part = unit % SPLITS * kFewDownWarps + warp, pieces = SPLITS * kFewDownWarps;
    const int begin = L.I / 16 * part / pieces, end = L.I / 16 * (part + 1) / pieces;
    const __nv_bfloat16* rows = L.down + (static_cast<size_t>(few.e) * L.I + 4 * t) * L.H + h0 + 8 * g;
    for (int pass = 0; pass < count; pass += 8) {
      uint4 w[kFewDownAhead][4];
      auto fetch = [&](int i, int step) {
#pragma unroll
        for (int r = 0; r < 4; ++r) w[i][r] = load_stream16(rows + static_cast<size_t>(16 * step + r) * L.H);
      };
#pragma unroll
      for (int i = 0; i < kFewDownAhead; ++i)
        if (begin + i < end) fetch(i, begin + i);
      if (!waited) grid_dependency_wait();
      waited = true;
      const int pair = pair_at(few.mask, pass + g);
      const size_t at = static_cast<size_t>(max(pair, 0)) * L.I + 4 * t;
      float acc[4][4] = {};
      for (int from = begin; from < end; from += kFewDownAhead) {
        uint2 x[kFewDownAhead][2];
#pragma unroll
        for (int i = 0; i < kFewDownAhead; ++i) {
          const bool has = pair >= 0 && from + i < end;
          x[i][0] = has ? *reinterpret_cast<const uint2*>(s.activations + at + 16 * (from + i)) : make_uint2(0, 0);
          x[i][1] = has ? *reinterpret_cast<const uint2*>(s.rests + at + 16 * (from + i)) : make_uint2(0, 0);
        }
#pragma unroll
        for (int i = 0; i < kFewDownAhead; ++i) {
          const int step = from + i;
          if (step >= end) break;
          const uint2* b = x[i];
          const uint32_t* v[4] = {&w[i][0].x, &w[i][1].x, &w[i][2].x, &w[i][3].x};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = __byte_perm(v[0][j], v[1][j], 0x5410), a1 = __byte_perm(v[0][j], v[1][j], 0x7632);
            const uint32_t a2 = __byte_perm(v[2][j], v[3][j], 0x5410), a3 = __byte_perm(v[2][j], v[3][j], 0x7632);
            mma_bf16(acc[j], a0, a1, a2, a3, b[0].x, b[0].y);
            mma_bf16(acc[j], a0, a1, a2, a3, b[1].x, b[1].y);
          }
          if (step + kFewDownAhead < end) fetch(i, step + kFewDownAhead);
        }
      }
      __syncthreads();  // the parts before have been added
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float4* to = reinterpret_cast<float4*>(&parts[warp][2 * t + c][8 * g]);
        to[0] = make_float4(acc[0][c], acc[0][2 + c], acc[1][c], acc[1][2 + c]);
        to[1] = make_float4(acc[2][c], acc[2][2 + c], acc[3][c], acc[3][2 + c]);
      }
      __syncthreads();
      for (int i = tid; i < min(8, count - pass) * kFewDownColumns; i += kFewDownThreads) {
        const int place = i / kFewDownColumns, column = i % kFewDownColumns;
        float sum = parts[0][place][column];
#pragma unroll
        for (int j = 1; j < kFewDownWarps; ++j) sum += parts[j][place][column];
        total[pair_at(few.mask, pass + place)][column] = sum;
      }
    }
  }
  if (!waited) grid_dependency_wait();
  grid_dependency_release();
  if (tid < kFewPairs) weights[tid] = weight;
  __syncthreads();
  cluster_meet();
  constexpr int kShare = kFewDownColumns / kFewRanks;
  for (int i = tid; i < routes.tokens * kShare; i += kFewDownThreads) {
    const int token = i / kShare, column = rank * kShare + i % kShare;
    float sum = 0.0f;
    constexpr int kSlots = kFewRanks / SPLITS;  // whose parts are on their way together
    for (int from = 0; from < L.K; from += kSlots) {
      float v[kSlots][SPLITS];
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const int pair = token * L.K + from + j, unit = from + j < L.K ? units[pair] : -1;
#pragma unroll
        for (int part = 0; part < SPLITS; ++part)
          v[j][part] = unit >= 0 ? *of_rank(&total[pair][column], (unit + part) % kFewRanks) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const int pair = token * L.K + from + j;
        if (from + j >= L.K || units[pair] < 0) continue;
#pragma unroll
        for (int part = 1; part < SPLITS; ++part) v[j][0] += v[j][part];
        sum = __fmaf_rn(weights[pair], v[j][0], sum);
      }
    }
    out[static_cast<size_t>(token) * L.H + h0 + column] = __float2bfloat16_rn(sum);
  }
  cluster_meet();  // the others' shared memory has been read
}

#include "cfm_experts_tc.cuh"

// ---- mix -------------------------------------------------------------------------------------------
constexpr int kMixThreads = 256;
constexpr int kMixAhead = 8;  // slots whose sums are on their way

// grid (T, H / 1024 and the rest): four columns of a token per thread.  The routes are asked for before the sums are there,
// and the sums of several slots at a time (one slot after another: 9.6 us for 64 tokens).
__global__ void __launch_bounds__(kMixThreads) k_experts_mix(Experts L, Scratch s, Routes routes, __nv_bfloat16* out) {
  __shared__ float weights[32];
  __shared__ unsigned has;
  const int token = blockIdx.x, column = (blockIdx.y * kMixThreads + threadIdx.x) * 4;
  if (threadIdx.x < 32) {
    const int pair = token * L.K + threadIdx.x;
    const bool valid = static_cast<int>(threadIdx.x) < L.K && routes.expert(pair, L.K, L.E) >= 0;
    weights[threadIdx.x] = valid ? routes.weight(pair) : 0.0f;
    const unsigned mask = __ballot_sync(kFull, valid);
    if (threadIdx.x == 0) has = mask;
  }
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_release();
  if (column >= L.H) return;
  const float* from = s.sums + static_cast<size_t>(token) * L.K * L.H + column;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int first = 0; first < L.K; first += kMixAhead) {
    float4 v[kMixAhead];
#pragma unroll
    for (int k = 0; k < kMixAhead; ++k)
      if (has >> (first + k) & 1) v[k] = *reinterpret_cast<const float4*>(from + static_cast<size_t>(first + k) * L.H);
#pragma unroll
    for (int k = 0; k < kMixAhead; ++k) {
      if (!(has >> (first + k) & 1)) continue;
      const float w = weights[first + k];
      sum = make_float4(__fmaf_rn(w, v[k].x, sum.x), __fmaf_rn(w, v[k].y, sum.y), __fmaf_rn(w, v[k].z, sum.z),
                        __fmaf_rn(w, v[k].w, sum.w));
    }
  }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
  *reinterpret_cast<uint2*>(out + static_cast<size_t>(token) * L.H + column) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// ---- host ------------------------------------------------------------------------------------------
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

int check_experts(const cfm_experts* x) {
  if (!x) return CFM_E_NULL;
  if (x->hidden < 128 || x->hidden % 128 || x->width < 16 || x->width % 16 || x->experts < 1 ||
      x->experts > kMaxExperts || x->top_k < 1 || x->top_k > 32 || x->hidden > 65536 || x->width > 65536)
    return CFM_E_SHAPE;
  if (x->activation != CFM_ACT_SILU && x->activation != CFM_ACT_GELU_TANH) return CFM_E_UNSUPPORTED;
  return 0;
}

// Bytes, and the arrays where `base` is given.
int64_t lay_out(const cfm_experts* x, int64_t capacity, void* base, Scratch* s) {
  int64_t at = 0;
  uint8_t* from = static_cast<uint8_t*>(base);
  auto take = [&](auto** array, int64_t count) {
    if (s) *array = reinterpret_cast<std::remove_reference_t<decltype(*array)>>(from + at);
    at = align256(at + count * static_cast<int64_t>(sizeof(**array)));
  };
  Scratch none;
  Scratch* to = s ? s : &none;
  const int64_t pairs = capacity * x->top_k;
  take(&to->status, 4);
  take(&to->pairs, pairs);
  take(&to->tokens, pairs);
  take(&to->passes, std::min<int64_t>(x->experts, pairs) + pairs / kLeastPass);
  take(&to->counts, 4);
  take(&to->activations, pairs * x->width);
  take(&to->rests, pairs * x->width);
  take(&to->sums, pairs * x->hidden);
  return at;
}

int run_few(const Experts& L, const Scratch& s, const Routes& routes, const __nv_bfloat16* hidden, int busy,
            __nv_bfloat16* out, cudaStream_t stream) {
  const int64_t items = static_cast<int64_t>(busy) * (L.I / 8);
  launch_dependent(k_few_up, dim3(static_cast<unsigned>(std::min<int64_t>(items, 148 * kFewUpPerSm))), dim3(kFewUpThreads), 0, stream, L, s, routes, hidden);
  // Parts of an expert's channels.  One, two and four of them, us of a call: K = 1 of 16 experts of width 1024, one token 13.9, 11.6, 11.4,
  // 16 tokens 34.2, 33.5, 37.3; K = 2 of 8 of hidden 4096 and width 1408, one token 34.0, 26.4, 23.9, eight tokens 61.4, 64.2, 68.8;
  // K = 4 of 16 of width 512, one token 13.0, 12.5 (two), four tokens 20.6, 21.8.
  const auto down = L.K >= 3 ? k_few_down<1> : k_few_down<2>;
  launch_clusters(down, dim3(L.H / kFewDownColumns * kFewRanks), dim3(kFewDownThreads), 0, kFewRanks, stream, L, s, routes, out);
  return launched();
}

// The map of a matrix [rows, columns] in boxes of 64 columns and 64 rows, swizzled by 128 bytes.
int make_map(CUtensorMap* map, const void* data, int64_t rows, int64_t columns) {
  static const auto encode = [] {
    void* found = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      found = nullptr;
    return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(found);
  }();
  if (!encode) return static_cast<int>(cudaErrorNotSupported);
  const cuuint64_t sizes[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(columns) * 2};
  const cuuint32_t box[2] = {kTensorColumns, 64}, steps[2] = {1, 1};
  const CUresult code = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(data), sizes, strides, box, steps,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return code == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

// Pairs of a pass, for `busy` experts.  A second pass over an expert reads its weights again, from L2; a stage with room for
// more tokens leaves fewer stages in the ring.  us of a call, measured in turn at the clocks of a busy GPU, of passes of 16, 32, 64 and 128:
// 64 tokens of the 128-expert layer (4 per expert) 203, 198, 204, 213; 256 of 256 experts with a skewed router (8) 209, 177, 175, 181.  Of 64,
// 128, 144, 160 and 192: 400 of 64 experts of width 768 (50) 136, 141, 141, 141, 150; 1000 of 64 experts of width 1024 (125) 364, 272, 236,
// 226, 239; 3000 of those (375) 934, 604, 616, 663, 629; 1000 of 32 experts of hidden 1024 (250) 162, 149, 135, 140, 154.
int pass_pairs(int64_t pairs, int64_t busy) { return pairs <= 12 * busy ? 32 : pairs <= 40 * busy ? 64 : 144; }

template <int TOKENS>
int run_tensor(const Experts& L, const Scratch& s, const __nv_bfloat16* hidden, int64_t pairs, cudaStream_t stream) {
  using U = Tensor<TOKENS, false>;
  using D = Tensor<TOKENS, true>;
  CUtensorMap up, down;
  int code = make_map(&up, L.gate_up, static_cast<int64_t>(L.E) * 2 * L.I, L.H);
  if (!code) code = make_map(&down, L.down, static_cast<int64_t>(L.E) * L.I, L.H);
  if (!code) code = allow_everything<k_experts_tensor<TOKENS, false>>(false);
  if (!code) code = allow_everything<k_experts_tensor<TOKENS, true>>(false);
  if (code) return code;
  const int64_t passes = std::min<int64_t>(L.E, pairs) + pairs / TOKENS;
  const auto ctas = [&](int tiles) { return dim3(static_cast<unsigned>(std::min<int64_t>(148, passes * tiles))); };
  launch_dependent(k_experts_tensor<TOKENS, false>, ctas((L.I + kUpTile - 1) / kUpTile), dim3(U::kThreads), U::kShared,
                   stream, L, s, hidden, up);
  launch_dependent(k_experts_tensor<TOKENS, true>, ctas(L.H / kTensorRows), dim3(D::kThreads), D::kShared, stream, L, s,
                   hidden, down);
  return 0;
}

}  // namespace
}  // namespace cfm

using namespace cfm;

extern "C" {

int64_t cfm_experts_workspace_bytes(const cfm_experts* layer, int32_t capacity) {
  const int code = check_experts(layer);
  if (code) return code;
  if (capacity < 1 || static_cast<int64_t>(capacity) * layer->top_k >= kMostPairs) return CFM_E_CAPACITY;
  return lay_out(layer, capacity, nullptr, nullptr);
}

int cfm_experts_forward(const cfm_experts* layer, void* workspace, int32_t capacity, const cfm_call* call, void* stream) {
  const int64_t bytes = cfm_experts_workspace_bytes(layer, capacity);
  if (bytes < 0) return static_cast<int>(bytes);
  if (!call || !workspace || !layer->gate_up || !layer->down || !call->hidden || !call->ids || !call->weights || !call->out)
    return CFM_E_NULL;
  if (call->tokens < 1 || call->tokens > capacity) return CFM_E_CAPACITY;
  for (const void* p : {layer->gate_up, layer->down, call->hidden, static_cast<const void*>(call->out), static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return CFM_E_SHAPE;
  Scratch s;
  lay_out(layer, capacity, workspace, &s);
  const Experts L = {layer->hidden, layer->width, layer->experts, layer->top_k, layer->activation,
                     static_cast<const __nv_bfloat16*>(layer->gate_up), static_cast<const __nv_bfloat16*>(layer->down)};
  const Routes routes = {call->ids, call->weights, call->padding, call->tokens, call->ids_are_int64, call->weights_are_bf16};
  const auto* hidden = static_cast<const __nv_bfloat16*>(call->hidden);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t pairs = static_cast<int64_t>(L.K) * call->tokens;
  const int busy = static_cast<int>(std::min<int64_t>(L.E, pairs));
  auto* out = static_cast<__nv_bfloat16*>(call->out);
  if (pairs <= kFewPairs) return run_few(L, s, routes, hidden, busy, out, st);
  if (const int code = allow_everything<k_group_pairs>(false)) return code;
  const int pass = pass_pairs(pairs, busy);
  launch_dependent(k_group_pairs, dim3(1), dim3(kGroupThreads), sizeof(int) * (L.E + kGroupKept * kGroupThreads), st,
                   routes, L.E, L.K, pass, s);
  const int code = pass == 32   ? run_tensor<32>(L, s, hidden, pairs, st)
                   : pass == 64 ? run_tensor<64>(L, s, hidden, pairs, st)
                                : run_tensor<144>(L, s, hidden, pairs, st);
  if (code) return code;
  launch_dependent(k_experts_mix, dim3(call->tokens, (L.H + 4 * kMixThreads - 1) / (4 * kMixThreads)), dim3(kMixThreads), 0,
                   st, L, s, routes, out);
  return launched();
}

}  // extern "C"
