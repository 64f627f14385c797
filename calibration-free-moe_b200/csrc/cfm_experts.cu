// The routed experts of one MoE layer as a whole (sm_100a): for every token the router-weighted sum over its
// experts of D_e (phi(G_e x) * (U_e x)), all channels, from the weights as the sparse reader keeps them.
//
// A call is bound by the weights of the experts that some token is routed to, so the (token, slot) pairs are
// grouped by expert and each weight is read once for all tokens of its expert:
//   group   counts, offsets and the list of pairs by expert
//   up      gate and up rows, activation, two BF16 terms [pair, I]
//   down    channel-major down rows, FP32 [pair, H]
//   mix     router weights, sum over a token's slots in their order, BF16
// Sums are FP32.  The tensor cores take the type of the weights, so an activation goes to them as two BF16
// terms, its value rounded and what that leaves: 2^-17 of it is lost, and of the output's error of 2^-9 nothing is theirs.
// (Rounded once to BF16 they would have added as much as the output's own rounding: 0.0024 of the output's norm
// instead of 0.0016.)
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
constexpr int kMaxWidth = 4096;  // eight tokens' activations fit shared memory

struct Experts {
  int H, I, E, K, activation;
  const __nv_bfloat16* gate_up;  // [E, 2 I, H]
  const __nv_bfloat16* down;     // [E, I, H]
};

struct Scratch {
  int32_t* offsets;  // [E + 1] first pair of every expert
  int32_t* pairs;    // [C K] pairs by expert
  int32_t* tokens;   // [C K] their tokens
  int32_t* busy;     // [E] experts that have pairs
  int4* passes;      // expert, first pair, pairs: of the tensor-core path
  int32_t* counts;   // [4] number of busy experts, of passes
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

  // The expert of a pair, -1 where it has none.
  __device__ int expert(int pair, int K, int E) const {
    if (padding && padding[pair / K]) return -1;
    const int64_t e = ids64 ? static_cast<const int64_t*>(ids)[pair] : static_cast<const int32_t*>(ids)[pair];
    return e >= 0 && e < E ? static_cast<int>(e) : -1;
  }
  __device__ float weight(int pair) const {
    return weights16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(weights)[pair])
                     : static_cast<const float*>(weights)[pair];
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
// and the three sums are scanned as one number.  The order of an expert's pairs is as it comes.
constexpr int kGroupThreads = 1024;
constexpr int kGroupKept = 8;  // pairs of a thread that stay in registers; of larger calls the rest is looked at twice
constexpr int64_t kMostPairs = 1 << 24;

// `tokens`: pairs of a pass.
__global__ void __launch_bounds__(kGroupThreads) k_group_pairs(Routes routes, int E, int K, int tokens, Scratch s) {
  extern __shared__ int group_shared[];
  __shared__ uint64_t warps[32];
  int* count = group_shared;  // [E], then the first place of every expert
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
  for (int p = tid + kGroupKept * kGroupThreads; p < pairs; p += kGroupThreads) {
    const int e = routes.expert(p, K, E);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  // Pairs, passes and busy experts before those of this thread, in one number.
  constexpr int kPassBits = 24, kBusyBits = kPassBits + 22;
  const int per = (E + kGroupThreads - 1) / kGroupThreads, from = min(E, tid * per), to = min(E, from + per);
  uint64_t mine = 0;
  for (int e = from; e < to; ++e)
    if (const int n = count[e])
      mine += static_cast<uint64_t>(n) | static_cast<uint64_t>((n + tokens - 1) / tokens) << kPassBits | 1ull << kBusyBits;
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
  const uint64_t before = sum - mine + (tid >= 32 ? warps[(tid >> 5) - 1] : 0), all = warps[31];
  int offset = static_cast<int>(before & ((1u << kPassBits) - 1)), part = static_cast<int>(before >> kPassBits & ((1u << 22) - 1));
  int place = static_cast<int>(before >> kBusyBits);
  for (int e = from; e < to; ++e) {
    const int n = count[e];
    s.offsets[e] = offset;
    count[e] = offset;
    for (int at = 0; at < n; at += tokens) s.passes[part++] = make_int4(e, offset + at, min(tokens, n - at), 0);
    offset += n;
    if (n) s.busy[place++] = e;
  }
  if (tid == 0) {
    s.offsets[E] = static_cast<int>(all & ((1u << kPassBits) - 1));
    s.counts[0] = static_cast<int>(all >> kBusyBits);
    s.counts[1] = static_cast<int>(all >> kPassBits & ((1u << 22) - 1));
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroupKept; ++j) {
    if (expert[j] < 0) continue;
    const int p = tid + j * kGroupThreads, at = count[expert[j]] + rank[j];
    s.pairs[at] = p;
    s.tokens[at] = p / K;
  }
  if (pairs <= kGroupKept * kGroupThreads) return;
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

// ---- up --------------------------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kSplits = 4;             // of a sum, over the warps of a CTA
constexpr int kUpChannels = 16;        // of a CTA: two warps' tiles of eight gate and eight up rows
constexpr int kUpAhead = 4;            // steps of 32 columns whose rows are on their way

// Tokens of a pass, columns of x in shared memory at a time.
template <int TILES>
struct Up {
  static constexpr int kTokens = 8 * TILES;
  static constexpr int kColumns = 4096 / TILES;
  static constexpr int kStride = 2 * kColumns + 64;  // bytes; rows of eight tokens fall into different banks
  static constexpr size_t kBytes = static_cast<size_t>(kTokens) * kStride;
  static constexpr size_t kSums = static_cast<size_t>(kThreads) * 4 * TILES * sizeof(float);
  static_assert(kSums <= kBytes, "the sums take the place of x");
};

// grid (I / 16, experts that can have pairs).  Weights go from global memory into the registers of the tensor
// cores' first operand as they lie: a thread has 16 bytes of a gate row and of an up row, whose
// elements are the k of two instructions, in an order that x is read in too.  Gate and up of a channel end in
// one thread.
template <int TILES>
__global__ void __launch_bounds__(kThreads, 2)
    k_experts_up(Experts L, Scratch s, const __nv_bfloat16* hidden) {
  using U = Up<TILES>;
  extern __shared__ __align__(16) uint8_t up_shared[];
  grid_dependency_wait();
  grid_dependency_release();
  if (static_cast<int>(blockIdx.y) >= s.counts[0]) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int split = warp & (kSplits - 1), tile = warp / kSplits;
  const int e = s.busy[blockIdx.y], first = s.offsets[e], pairs = s.offsets[e + 1] - first;
  const int c0 = blockIdx.x * kUpChannels;
  const __nv_bfloat16* gate = L.gate_up + (static_cast<size_t>(e) * 2 * L.I + c0 + 8 * tile + g) * L.H + 8 * t;
  const __nv_bfloat16* up = gate + static_cast<size_t>(L.I) * L.H;

  for (int pass = 0; pass < pairs; pass += U::kTokens) {
    const int tokens = min(U::kTokens, pairs - pass);
    float acc[TILES][4] = {};
    for (int k0 = 0; k0 < L.H; k0 += U::kColumns) {
      const int columns = min(U::kColumns, L.H - k0), steps = columns / (32 * kSplits);
      const size_t at = k0 + 32 * split;  // a warp's steps lie 128 columns apart, whatever the passes are
      uint4 a[kUpAhead], b[kUpAhead];
#pragma unroll
      for (int i = 0; i < kUpAhead; ++i)
        if (i < steps) {
          a[i] = load_stream16(gate + at + 128 * i);
          b[i] = load_stream16(up + at + 128 * i);
        }
      __syncthreads();  // the columns before have been read
      for (int i = tid; i < tokens * (columns / 8); i += kThreads) {
        const int row = i / (columns / 8), piece = i - row * (columns / 8);
        const int token = s.tokens[first + pass + row];
        copy_async16(shared_u32(up_shared + row * U::kStride + 16 * piece),
                     hidden + static_cast<size_t>(token) * L.H + k0 + 8 * piece);
      }
      copy_async_commit();
      copy_async_wait<0>();
      __syncthreads();
      const uint32_t x = shared_u32(up_shared) + g * U::kStride + 64 * split + 16 * t;
      for (int from = 0; from < steps; from += kUpAhead) {
#pragma unroll
        for (int i = 0; i < kUpAhead; ++i) {
          if (from + i >= steps) break;
          const uint4 ga = a[i], ua = b[i];
          if (from + i + kUpAhead < steps) {
            a[i] = load_stream16(gate + at + 128 * (from + i + kUpAhead));
            b[i] = load_stream16(up + at + 128 * (from + i + kUpAhead));
          }
#pragma unroll
          for (int n = 0; n < TILES; ++n) {
            const uint4 v = load_shared16(x + n * 8 * U::kStride + 256 * (from + i));
            mma_bf16(acc[n], ga.x, ua.x, ga.y, ua.y, v.x, v.y);
            mma_bf16(acc[n], ga.z, ua.z, ga.w, ua.w, v.z, v.w);
          }
        }
      }
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(up_shared);  // [tile of channels][split][token tile][4][lane]
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[((warp * TILES + n) * 4 + i) * 32 + lane] = acc[n][i];
    __syncthreads();
    for (int i = tid; i < kUpChannels * 8 * TILES; i += kThreads) {
      const int c = i % kUpChannels, token = i / kUpChannels;
      if (token >= tokens) continue;
      const int from_lane = (c & 7) * 4 + ((token & 7) >> 1);
      float gu[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float* of = sums + ((c / 8 * kSplits * TILES + token / 8) * 4 + 2 * half + (token & 1)) * 32 + from_lane;
        float sum = of[0];
#pragma unroll
        for (int j = 1; j < kSplits; ++j) sum += of[j * TILES * 128];
        gu[half] = sum;
      }
      store_activation(s, static_cast<size_t>(s.pairs[first + pass + token]) * L.I + c0 + c,
                       gated(gu[0], gu[1], L.activation));
    }
    __syncthreads();
  }
}

// ---- down ------------------------------------------------------------------------------------------
constexpr int kDownColumns = 128;  // of a CTA: two warps' 64
constexpr int kDownAhead = 2;      // steps of 16 channels whose rows are on their way

// grid (H / 128, experts that can have pairs).  A thread has 16 bytes, eight outputs, of four channels' rows; the
// first operand's registers pair two channels of one output, which two byte permutations per pair of words do.
template <int TILES>
__global__ void __launch_bounds__(kThreads, 2) k_experts_down(Experts L, Scratch s) {
  extern __shared__ __align__(16) uint8_t down_shared[];
  grid_dependency_wait();
  grid_dependency_release();
  if (static_cast<int>(blockIdx.y) >= s.counts[0]) return;
  constexpr int kTokens = 8 * TILES;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int split = warp & (kSplits - 1), half = warp / kSplits;
  const int e = s.busy[blockIdx.y], first = s.offsets[e], pairs = s.offsets[e + 1] - first;
  const int h0 = blockIdx.x * kDownColumns + 64 * half;
  const int all = L.I / 16, begin = all * split / kSplits, end = all * (split + 1) / kSplits;
  const int stride = (2 * L.I + 127) / 128 * 128 + 32;  // bytes of a row of activations
  const __nv_bfloat16* rows = L.down + (static_cast<size_t>(e) * L.I + 4 * t) * L.H + h0 + 8 * g;
  auto fetch = [&](uint4 (&w)[4], int step) {
#pragma unroll
    for (int r = 0; r < 4; ++r) w[r] = load_stream16(rows + static_cast<size_t>(16 * step + r) * L.H);
  };

  for (int pass = 0; pass < pairs; pass += kTokens) {
    const int tokens = min(kTokens, pairs - pass);
    uint4 w[kDownAhead][4];
#pragma unroll
    for (int i = 0; i < kDownAhead; ++i)
      if (begin + i < end) fetch(w[i], begin + i);
    __syncthreads();
    for (int i = tid; i < tokens * (L.I / 8); i += kThreads) {
      const int row = i / (L.I / 8), piece = i - row * (L.I / 8);
      const size_t from = static_cast<size_t>(s.pairs[first + pass + row]) * L.I + 8 * piece;
      copy_async16(shared_u32(down_shared + row * stride + 16 * piece), s.activations + from);
      copy_async16(shared_u32(down_shared + (kTokens + row) * stride + 16 * piece), s.rests + from);
    }
    copy_async_commit();
    copy_async_wait<0>();
    __syncthreads();
    float acc[TILES][4][4] = {};
    const uint32_t x = shared_u32(down_shared) + g * stride + 8 * t;
    for (int from = begin; from < end; from += kDownAhead) {
#pragma unroll
      for (int i = 0; i < kDownAhead; ++i) {
        const int step = from + i;
        if (step >= end) break;
        uint32_t a[4][4];
        const uint32_t* v[4] = {&w[i][0].x, &w[i][1].x, &w[i][2].x, &w[i][3].x};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[j][0] = __byte_perm(v[0][j], v[1][j], 0x5410);
          a[j][1] = __byte_perm(v[0][j], v[1][j], 0x7632);
          a[j][2] = __byte_perm(v[2][j], v[3][j], 0x5410);
          a[j][3] = __byte_perm(v[2][j], v[3][j], 0x7632);
        }
        if (step + kDownAhead < end) fetch(w[i], step + kDownAhead);
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            uint32_t b0, b1;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                         : "=r"(b0), "=r"(b1)
                         : "r"(x + (term * kTokens + n * 8) * stride + 32 * step));
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_bf16(acc[n][j], a[j][0], a[j][1], a[j][2], a[j][3], b0, b1);
          }
        }
      }
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(down_shared);  // [half][split][token][64]
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float4* to = reinterpret_cast<float4*>(sums + (static_cast<size_t>(warp) * kTokens + 8 * n + 2 * t + c) * 64 + 8 * g);
        to[0] = make_float4(acc[n][0][c], acc[n][0][2 + c], acc[n][1][c], acc[n][1][2 + c]);
        to[1] = make_float4(acc[n][2][c], acc[n][2][2 + c], acc[n][3][c], acc[n][3][2 + c]);
      }
    __syncthreads();
    for (int i = tid; i < tokens * (kDownColumns / 4); i += kThreads) {
      const int token = i / (kDownColumns / 4), column = i % (kDownColumns / 4) * 4;
      const float* of = sums + (static_cast<size_t>(column / 64 * kSplits) * kTokens + token) * 64 + column % 64;
      float4 sum = *reinterpret_cast<const float4*>(of);
#pragma unroll
      for (int j = 1; j < kSplits; ++j) {
        const float4 more = *reinterpret_cast<const float4*>(of + static_cast<size_t>(j) * kTokens * 64);
        sum = make_float4(sum.x + more.x, sum.y + more.y, sum.z + more.z, sum.w + more.w);
      }
      const int pair = s.pairs[first + pass + token];
      *reinterpret_cast<float4*>(s.sums + static_cast<size_t>(pair) * L.H + blockIdx.x * kDownColumns + column) = sum;
    }
    __syncthreads();
  }
}

template <int TILES>
static size_t down_shared_bytes(int I) {
  const size_t rows = 2 * 8 * TILES * static_cast<size_t>((2 * I + 127) / 128 * 128 + 32);
  return std::max(rows, static_cast<size_t>(kThreads / 32) * 8 * TILES * 64 * sizeof(float));
}

#include "cfm_experts_tc.cuh"

// ---- mix -------------------------------------------------------------------------------------------
constexpr int kMixThreads = 128;

// grid (T, H / 1024 and the rest): eight columns of a token per thread.
__global__ void __launch_bounds__(kMixThreads) k_experts_mix(Experts L, Scratch s, Routes routes, __nv_bfloat16* out) {
  grid_dependency_wait();
  grid_dependency_release();
  const int token = blockIdx.x, column = (blockIdx.y * kMixThreads + threadIdx.x) * 8;
  if (column >= L.H) return;
  float sum[8] = {};
  for (int k = 0; k < L.K; ++k) {
    const int pair = token * L.K + k;
    if (routes.expert(pair, L.K, L.E) < 0) continue;
    const float w = routes.weight(pair);
    const float4* from = reinterpret_cast<const float4*>(s.sums + static_cast<size_t>(pair) * L.H + column);
    const float4 a = from[0], b = from[1];
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = __fmaf_rn(w, v[i], sum[i]);
  }
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(sum[2 * i], sum[2 * i + 1]);
    words[i] = *reinterpret_cast<const uint32_t*>(&pair);
  }
  *reinterpret_cast<uint4*>(out + static_cast<size_t>(token) * L.H + column) =
      make_uint4(words[0], words[1], words[2], words[3]);
}

// ---- host ------------------------------------------------------------------------------------------
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

int check_experts(const cfm_experts* x) {
  if (!x) return CFM_E_NULL;
  if (x->hidden < 128 || x->hidden % 128 || x->width < 16 || x->width % 16 || x->experts < 1 ||
      x->experts > kMaxExperts || x->top_k < 1 || x->top_k > 32 || x->hidden > 65536 || x->width > kMaxWidth)
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
  take(&to->offsets, x->experts + 1);
  take(&to->pairs, pairs);
  take(&to->tokens, pairs);
  take(&to->busy, x->experts);
  take(&to->passes, std::min<int64_t>(x->experts, pairs) + pairs / kLeastPass);
  take(&to->counts, 4);
  take(&to->activations, pairs * x->width);
  take(&to->rests, pairs * x->width);
  take(&to->sums, pairs * x->hidden);
  return at;
}

template <typename K>
int allow_shared(K kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return 0;
  return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

template <int TILES>
int run_tiles(const Experts& L, const Scratch& s, const __nv_bfloat16* hidden, int busy, cudaStream_t stream) {
  const size_t down = down_shared_bytes<TILES>(L.I);
  int code = allow_shared(k_experts_up<TILES>, Up<TILES>::kBytes);
  if (!code) code = allow_shared(k_experts_down<TILES>, down);
  if (code) return code;
  launch_dependent(k_experts_up<TILES>, dim3(L.I / kUpChannels, busy), dim3(kThreads), Up<TILES>::kBytes, stream, L, s, hidden);
  launch_dependent(k_experts_down<TILES>, dim3(L.H / kDownColumns, busy), dim3(kThreads), down, stream, L, s);
  return 0;
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

// Pairs of a pass, for `busy` experts.  A second pass over an expert reads its weights again, from L2; a stage with room for more
// tokens leaves fewer stages in the ring.  Passes of 16, 32, 64, 128 (and 192), us of a call: 64 tokens of the
// 128-expert layer (4 per expert) 200, 195, 196, 205; 256 of 256 experts with a skewed router (8) 192, 168, 168, 169;
// 1000 of 64 experts (125) 828, 452, 299, 234, 216.
int pass_pairs(int64_t pairs, int64_t busy) {
  return pairs <= 12 * busy ? 32 : pairs <= 32 * busy ? 64 : pairs <= 80 * busy ? 128 : 192;
}

template <int TOKENS>
int run_tensor(const Experts& L, const Scratch& s, const __nv_bfloat16* hidden, int64_t pairs, cudaStream_t stream) {
  using U = Tensor<TOKENS, false>;
  using D = Tensor<TOKENS, true>;
  CUtensorMap up, down;
  int code = make_map(&up, L.gate_up, static_cast<int64_t>(L.E) * 2 * L.I, L.H);
  if (!code) code = make_map(&down, L.down, static_cast<int64_t>(L.E) * L.I, L.H);
  if (!code) code = allow_shared(k_experts_tensor<TOKENS, false>, U::kShared);
  if (!code) code = allow_shared(k_experts_tensor<TOKENS, true>, D::kShared);
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
  Scratch s;
  lay_out(layer, capacity, workspace, &s);
  const Experts L = {layer->hidden, layer->width, layer->experts, layer->top_k, layer->activation,
                     static_cast<const __nv_bfloat16*>(layer->gate_up), static_cast<const __nv_bfloat16*>(layer->down)};
  const Routes routes = {call->ids, call->weights, call->padding, call->tokens, call->ids_are_int64, call->weights_are_bf16};
  const auto* hidden = static_cast<const __nv_bfloat16*>(call->hidden);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t pairs = static_cast<int64_t>(L.K) * call->tokens;
  const int busy = static_cast<int>(std::min<int64_t>(L.E, pairs));
  const int pass = pass_pairs(pairs, busy);
  launch_dependent(k_group_pairs, dim3(1), dim3(kGroupThreads), sizeof(int) * L.E, st, routes, L.E, L.K, pass, s);
  const int code = pairs <= 32    ? run_tiles<1>(L, s, hidden, busy, st)
                   : pass == 32   ? run_tensor<32>(L, s, hidden, pairs, st)
                   : pass == 64   ? run_tensor<64>(L, s, hidden, pairs, st)
                   : pass == 128  ? run_tensor<128>(L, s, hidden, pairs, st)
                                  : run_tensor<192>(L, s, hidden, pairs, st);
  if (code) return code;
  launch_dependent(k_experts_mix, dim3(call->tokens, (L.H + 8 * kMixThreads - 1) / (8 * kMixThreads)), dim3(kMixThreads), 0,
                   st, L, s, routes, static_cast<__nv_bfloat16*>(call->out));
  return launched();
}

}  // extern "C"
