// Operators over rows of logits (sm_100a): the router's softmax and top-k, log probabilities of given
// tokens with entropy and top alternatives, and the divergence of two rows of logits.
//
// Rows are of BF16, FP16 or FP32, any number of elements apart and at any element's alignment.  All
// arithmetic is in FP32 or more.  The order of values is total wherever one is picked: larger first, NaN
// above all, equal ones (0 and -0 among them) by the lowest index; so nothing depends on how a row is split.
#include "cfm_device.cuh"
#include "cfm_launch.cuh"

#include "cfm_b200.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace cfm {

typedef unsigned long long u64;

constexpr float kLog2E = 1.44269504f;
constexpr float kInfinity = __builtin_huge_valf();
// Stands for -inf where sums want a finite number: beside a largest value of up to kModerate its exponential is zero.
constexpr float kLeast = -1e30f, kModerate = 1e29f;
// Largest size of a shift m for which m log2 e may be rounded: by half a unit of the last place, 64 at most, which powers
// of two make good, for logits of such a size are no closer to each other.  (With 2^24, the divergence of rows masked by
// -1e9 took 14 % longer.)
constexpr float kScaled = 1073741824.0f;

// 2^x, two units in the last place; 0 below -126.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^d.  The product is rounded apart, so that its error is of d and not of a larger number's.
__device__ __forceinline__ float exp_fast(float d) { return exp2_fast(__fmul_rn(d, kLog2E)); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float warp_max_nan(float x) {
  float y;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Unsigned integers in the order of the values; 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(__fadd_rn(x, 0.0f));  // -0 becomes 0
  if (x != x) return 0xffffffffu;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return key == 0xffffffffu ? __int_as_float(0x7fffffff)
                            : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// A value with its place; no two are equal, and the lower place of two equal values is the larger one.
__device__ __forceinline__ u64 placed(float x, uint32_t index) {
  return static_cast<u64>(ordered(x)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int place_of(u64 key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

__device__ __forceinline__ u64 shuffle_xor(u64 v, int mask) { return __shfl_xor_sync(kFull, v, mask); }

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int w = 16; w; w >>= 1) v = max(v, shuffle_xor(v, w));
  return v;
}

// The warp's values in descending order.  (Not inlined, as other parts that run once or twice per CTA are not: code that
// is met for the first time comes from L2, and that was half of a call of one token.)
__device__ __noinline__ u64 warp_sort(u64 v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int w = size >> 1; w; w >>= 1) {
      const u64 other = shuffle_xor(v, w);
      const bool larger_first = (lane & size) == 0 || size == 32;
      const bool keep_larger = ((lane & w) == 0) == larger_first;
      v = keep_larger ? max(v, other) : min(v, other);
    }
  return v;
}
// The largest 32 of two lists in descending order, in descending order: of a list and the other one
// backwards the larger ones are those, as a bitonic sequence.
__device__ __noinline__ u64 warp_merge(u64 a, u64 b, int lane) {
  u64 v = max(a, __shfl_sync(kFull, b, 31 - lane));
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    const u64 other = shuffle_xor(v, w);
    v = (lane & w) == 0 ? max(v, other) : min(v, other);
  }
  return v;
}

// ---- rows ------------------------------------------------------------------------------------------
template <typename T>
struct Element;
template <>
struct Element<__nv_bfloat16> {
  static constexpr int kWidth = 8;
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static void widen(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  // Largest value of pieces, NaN if one is.
  using Top = uint32_t;
  static constexpr uint32_t kNone = 0xff80ff80u;
  __device__ static Top lowest() { return kNone; }
  __device__ static void fold(Top& top, const uint4& v) {
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v.x));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v.y));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v.z));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v.w));
  }
  __device__ static float value(Top top) { return max_nan(bf16_lo(top), bf16_hi(top)); }
  // With -inf (and NaN) raised to kLeast.
  __device__ static void widen_bounded(uint4 v, float* x) {
    constexpr uint32_t least = 0xf149f149u;  // twice, rounded down
    asm("max.bf16x2 %0, %0, %1;" : "+r"(v.x) : "r"(least));
    asm("max.bf16x2 %0, %0, %1;" : "+r"(v.y) : "r"(least));
    asm("max.bf16x2 %0, %0, %1;" : "+r"(v.z) : "r"(least));
    asm("max.bf16x2 %0, %0, %1;" : "+r"(v.w) : "r"(least));
    widen(v, x);
  }
  __device__ static float largest(const uint4& v) {
    uint32_t a, b;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return max_nan(bf16_lo(a), bf16_hi(a));
  }
};
template <>
struct Element<__half> {
  static constexpr int kWidth = 8;
  __device__ static float one(const __half* p) { return __half2float(*p); }
  __device__ static void widen(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  using Top = uint32_t;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  __device__ static Top lowest() { return kNone; }
  __device__ static void fold(Top& top, const uint4& v) {
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(v.x));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(v.y));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(v.z));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(v.w));
  }
  __device__ static float value(Top top) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&top));
    return max_nan(f.x, f.y);
  }
  __device__ static void widen_bounded(const uint4& v, float* x) {
    widen(v, x);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) x[i] = fmaxf(x[i], kLeast);
  }
  __device__ static float largest(const uint4& v) {
    uint32_t a, b;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
    return max_nan(f.x, f.y);
  }
};
template <>
struct Element<float> {
  static constexpr int kWidth = 4;
  __device__ static float one(const float* p) { return *p; }
  __device__ static void widen(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  using Top = float;
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ static Top lowest() { return -kInfinity; }
  __device__ static void fold(Top& top, const uint4& v) { top = max_nan(top, largest(v)); }
  __device__ static float value(Top top) { return top; }
  __device__ static void widen_bounded(const uint4& v, float* x) {
    widen(v, x);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) x[i] = fmaxf(x[i], kLeast);
  }
  __device__ static float largest(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                   max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};

// A row as 16-byte pieces: the first and the last one may reach over its ends, where nothing is read.
// Where two rows are read together they may be aligned differently, so a piece has the elements
// [W v - shift, W v - shift + W) of its row and is read whole only where it lies on a 16-byte boundary.
template <typename T>
struct Row {
  static constexpr int W = Element<T>::kWidth;
  const T* data;
  int columns, shift;
  bool aligned;  // whole pieces lie on 16-byte boundaries

  __device__ Row(const void* rows, int64_t stride, int64_t row, int columns_, int shift_ = -1)
      : data(static_cast<const T*>(rows) + row * stride), columns(columns_) {
    const int past = static_cast<int>((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
    shift = shift_ < 0 ? past : shift_;
    aligned = past == shift;
  }
  __device__ int pieces() const { return (columns + shift + W - 1) / W; }
  __device__ int first(int piece) const { return piece * W - shift; }
  __device__ bool whole(int piece) const {
    const int at = first(piece);
    return aligned && at >= 0 && at + W <= columns;
  }
  // -inf stands where the row has nothing.
  __device__ uint4 load(int piece) const {
    if (whole(piece)) return __ldg(reinterpret_cast<const uint4*>(data + first(piece)));
    return load_edge(data, first(piece), columns);
  }
  __device__ __noinline__ static uint4 load_edge(const T* data, int at, int columns) {
    union {
      T e[W];
      uint4 v;
    } u;
    u.v = make_uint4(Element<T>::kNone, Element<T>::kNone, Element<T>::kNone, Element<T>::kNone);
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (at + i >= 0 && at + i < columns) u.e[i] = data[at + i];
    return u.v;
  }
};

// ---- router ----------------------------------------------------------------------------------------
constexpr int kRouteRows = 4;       // a warp each
constexpr int kRouteColumns = 1024;

// K maxima one after another by a warp; lanes hold columns 32 apart.  What a row costs is latency: two
// reductions of the warp per expert picked.
template <typename T, int PER>
__global__ void __launch_bounds__(32 * kRouteRows)
    k_route_tokens(const void* logits, int64_t stride, int rows, int E, int K, int renormalize, void* ids,
                   int ids64, void* weights, int weights16) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRouteRows + (threadIdx.x >> 5);
  grid_dependency_wait();
  grid_dependency_release();
  if (row >= rows) return;
  const T* x = static_cast<const T*>(logits) + row * stride;
  float value[PER];
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    value[i] = e < E ? Element<T>::one(x + e) : -kInfinity;
    key[i] = e < E ? ordered(value[i]) : 0;
  }
  int mine = 0;
  float weight = 0.0f, largest = 0.0f, kept = 0.0f;
  for (int k = 0; k < K; ++k) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint32_t top = __reduce_max_sync(kFull, best);
    const int e = __reduce_min_sync(kFull, best == top ? static_cast<uint32_t>(lane + 32 * at) : 0xffffffffu);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e == lane + 32 * i) key[i] = 0;
    if (k == 0) largest = value_of(top);
    const float share = expf(value_of(top) - largest);
    kept += share;
    if (lane == k) {
      mine = e;
      weight = share;
    }
  }
  float total = kept;
  if (!renormalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < E) total += expf(value[i] - largest);
#pragma unroll
    for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(kFull, total, w);
  }
  if (lane >= K) return;
  weight = __fdiv_rn(weight, total);
  const int64_t at = row * K + lane;
  if (ids64) static_cast<int64_t*>(ids)[at] = mine;
  else static_cast<int32_t*>(ids)[at] = mine;
  if (weights16) static_cast<__nv_bfloat16*>(weights)[at] = __float2bfloat16_rn(weight);
  else static_cast<float*>(weights)[at] = weight;
}

// ---- log probabilities -----------------------------------------------------------------------------
constexpr int kScoreThreads = 256;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScorePerSm = 4;
constexpr int kScorePieces = 3;                 // of a thread that are added up together
constexpr int kScoreChunks = 2;                 // of so many pieces that are on their way or kept
constexpr int kScoreRing = kScoreChunks * kScorePieces;
constexpr size_t kRingBytes = static_cast<size_t>(kScoreThreads) * kScoreRing * 16;
constexpr int kFound = 512;
constexpr int kChunksKnown = 64;                // whose largest values the second pass looks at
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 16;

// A thread's pieces of a row in shared memory, which it alone writes and reads.
__device__ __forceinline__ uint32_t ring_slot(uint32_t ring, int slot) {
  return ring + (slot * kScoreThreads + threadIdx.x) * 16;
}
__device__ __forceinline__ void store_shared16(uint32_t address, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Sums over elements x with the largest m: e^(x - m) without the `equal` elements that are m, and
// e^(x - m) (x - m).  Without them the sum keeps its digits where one token has nearly all probability:
// its log probability is then -log1p of the others' sum.
struct Sums {
  float m, equal, others, weighted;
};

// The sums of a lane's elements and of the other lanes', 2 * width of them, brought to one shift; every one of
// those lanes has it.
__device__ __noinline__ Sums sums_of_lanes(Sums s, int width) {
  float m = s.m;
  for (int w = width; w; w >>= 1) m = max_nan(m, __shfl_xor_sync(kFull, m, w));
  if (s.m != m) {  // -inf: has seen nothing else
    const float step = s.m - m, f = s.m > -kInfinity ? exp_fast(step) : 0.0f, all = s.others + s.equal;
    s.weighted = f > 0.0f ? f * (s.weighted + step * all) : 0.0f;
    s.others = f * all;
    s.equal = 0.0f;
    s.m = m;
  }
  for (int w = width; w; w >>= 1) {
    s.equal += __shfl_xor_sync(kFull, s.equal, w);
    s.others += __shfl_xor_sync(kFull, s.others, w);
    s.weighted += __shfl_xor_sync(kFull, s.weighted, w);
  }
  return s;
}

// Tops of `count` descending lists of 32, twice the warps at most, in the first list; all threads.
__device__ __noinline__ void merge_lists(u64 (*lists)[32], int count, int warp, int lane) {
  for (int step = 1; step < count; step <<= 1) {
    __syncthreads();
    const int to = 2 * step * warp;
    if (to + step < count) lists[to][lane] = warp_merge(lists[to][lane], lists[to + step][lane], lane);
  }
  __syncthreads();
}

// One cluster per row; its CTAs share the row's pieces and hand their results to the first one.  One pass over the
// row gives the sums: per warp, with the warp's largest value so far as the shift.  The top alternatives take a second
// pass, from shared memory where the CTA's pieces fit the ring, else from the caches: the n-th largest of the
// threads' own maxima is not above the n-th largest element, so few elements are as large; those are sorted.  Should
// more than kFound be, the n-th largest of the first ones is a closer bound, and the pass is taken again: each time all but
// n of those are out.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, kScorePerSm)
    k_token_logprobs(const void* logits, int64_t stride, int V, const void* tokens, int tokens64, int n, float* logprobs,
                     float* entropy, int32_t* top_ids, float* top_logprobs) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  extern __shared__ __align__(16) uint8_t score_shared[];
  __shared__ u64 found[kFound], lists[kScoreWarps][32], ranked[kMaxCluster][32];
  __shared__ Sums sums[kScoreWarps], ranks_sums[kMaxCluster];
  __shared__ float s_log_z, s_m, chunk_tops[kScoreWarps][kChunksKnown];
  __shared__ int s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = cluster_size(), rank = cluster_rank();
  const int64_t r = blockIdx.x / ranks;
  const uint32_t ring = shared_u32(score_shared);
  cluster_arrive();
  grid_dependency_wait();
  grid_dependency_release();
  const Row<T> row(logits, stride, r, V);
  const int pieces = row.pieces();
  const int begin = static_cast<int>(static_cast<int64_t>(pieces) * rank / ranks);
  const int end = static_cast<int>(static_cast<int64_t>(pieces) * (rank + 1) / ranks);
  const bool kept = end - begin <= kScoreRing * kScoreThreads;
  // The thread's pieces are begin + tid, + 256, ...; a chunk is kScorePieces of them, of every thread.  -inf where it
  // has no more.
  constexpr int kChunk = kScorePieces * kScoreThreads;
  const int whole_from = row.whole(0) ? 0 : 1, whole_to = row.whole(pieces - 1) ? pieces : pieces - 1;
  auto bring_chunk = [&](int first, int slot) {
    if (first >= whole_from && first + kChunk <= min(end, whole_to)) {
      const T* from = row.data + row.first(first + tid);
#pragma unroll
      for (int j = 0; j < kScorePieces; ++j) copy_async16(ring_slot(ring, slot + j), from + j * kScoreThreads * W);
    } else {
#pragma unroll 1
      for (int j = 0; j < kScorePieces; ++j) {
        const int p = first + tid + j * kScoreThreads;
        if (p < end && row.whole(p)) copy_async16(ring_slot(ring, slot + j), row.data + row.first(p));
        else store_shared16(ring_slot(ring, slot + j), p < end ? row.load(p) : make_uint4(E::kNone, E::kNone, E::kNone, E::kNone));
      }
    }
    copy_async_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kScoreChunks; ++i) bring_chunk(begin + i * kChunk, kScorePieces * i);
  int64_t token = -1;
  if (rank == 0 && tid == 0)
    token = tokens64 ? static_cast<const int64_t*>(tokens)[r] : static_cast<const int32_t*>(tokens)[r];

  float best = -kInfinity;  // of the thread, NaN above all, and the first chunk that has it
  int best_chunk = begin;
  float m = -kInfinity, equal = 0.0f, others = 0.0f, weighted = 0.0f;
  int slot = 0, number = 0;
  for (int first = begin; first < end; first += kChunk, ++number) {
    copy_async_wait<kScoreChunks - 1>();
    uint4 v[kScorePieces];
    typename E::Top highest = E::lowest();
#pragma unroll
    for (int j = 0; j < kScorePieces; ++j) {
      v[j] = load_shared16(ring_slot(ring, slot + j));
      E::fold(highest, v[j]);
    }
    const float top = E::value(highest);
    if (!kept) bring_chunk(first + kScoreChunks * kChunk, slot);
    else copy_async_commit();
    slot = slot + kScorePieces == kScoreRing ? 0 : slot + kScorePieces;
    if (!(top <= best) && best == best) {
      best = top;
      best_chunk = first;
    }
    const float chunk = warp_max_nan(top);
    if (lane == 0 && number < kChunksKnown) chunk_tops[warp][number] = chunk;
    if (!(chunk <= m) && m == m) {  // a new shift, the same in the whole warp; NaN stays
      const float step = m - chunk, f = m == -kInfinity ? 0.0f : exp_fast(step);
      const float all = others + equal;
      weighted = f > 0.0f ? f * (weighted + step * all) : 0.0f;
      others = f * all;
      equal = 0.0f;
      m = chunk;
    }
    if (m == -kInfinity) continue;  // nothing but -inf so far
    if (fabsf(m) <= kScaled) {
      // In powers of two, from one multiply-add per element: 2^t, t = x log2 e - c, c = m log2 e as it rounds.
      // m itself has t = t_m, next to zero; with that the chunk's sums are brought to the shift m.
      const float c = __fmul_rn(m, kLog2E), t_m = __fmaf_rn(m, kLog2E, -c);
      const Pair scale = pair_of(kLog2E, kLog2E), shift = pair_of(-c, -c);
      Pair sum = pair_of(0.0f, 0.0f), moment = sum;
#pragma unroll
      for (int j = 0; j < kScorePieces; ++j) {
        float x[W];
        E::widen_bounded(v[j], x);
        if (top == m) {
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (x[i] == m) {
              equal += 1.0f;
              x[i] = kLeast;
            }
        }
#pragma unroll
        for (int i = 0; i < W; i += 2) {
          const Pair t = pair_fma(pair_of(x[i], x[i + 1]), scale, shift);
          float t0, t1;
          pair_split(t, t0, t1);
          const Pair e = pair_of(exp2_fast(t0), exp2_fast(t1));
          sum = pair_add(sum, e);
          moment = pair_fma(e, t, moment);
        }
      }
      float s0, s1, w0, w1;
      pair_split(sum, s0, s1);
      pair_split(moment, w0, w1);
      const float back = exp2_fast(-t_m), all = s0 + s1;
      others = __fmaf_rn(all, back, others);
      weighted = __fmaf_rn(0.693147181f * back, (w0 + w1) - t_m * all, weighted);
      continue;
    }
    // Larger ones (a mask of a finite value, mostly), or NaN, which the shift tells of.  (The same as above with m taken from the
    // elements first, by a test per piece: 39.2 us for 512 rows of 151936, against 38.4.)
#pragma unroll
    for (int j = 0; j < kScorePieces; ++j) {
      float x[W];
      E::widen(v[j], x);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float d = x[i] == m ? kLeast : fmaxf(__fsub_rn(x[i], m), kLeast);  // -inf: adds nothing
        const float e = exp_fast(d);
        equal += x[i] == m;
        others += e;
        weighted = __fmaf_rn(e, d, weighted);
      }
    }
  }
  const bool given = token >= 0 && token < V;
  const float x_token = given ? E::one(row.data + token) : 0.0f;
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    equal += __shfl_xor_sync(kFull, equal, w);
    others += __shfl_xor_sync(kFull, others, w);
    weighted += __shfl_xor_sync(kFull, weighted, w);
  }
  if (lane == 0) sums[warp] = {m, equal, others, weighted};

  if (n) {
    // The thread's largest element, NaN above all.
    auto again = [&](int p) { return kept ? load_shared16(ring_slot(ring, (p - begin) / kScoreThreads)) : row.load(p); };
    int best_piece = -1;
#pragma unroll 1
    for (int p = best_chunk + tid; p < min(end, best_chunk + kChunk) && best_piece < 0; p += kScoreThreads) {
      const float highest = E::largest(again(p));
      if (highest == best || (highest != highest && best != best)) best_piece = p;
    }
    u64 top = 0;
    if (best_piece >= 0) {
      float x[W];
      E::widen(again(best_piece), x);
      const int at = row.first(best_piece);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (at + i >= 0 && at + i < V) top = max(top, placed(x[i], at + i));
    }
    lists[warp][lane] = warp_sort(top, lane);
    merge_lists(lists, kScoreWarps, warp, lane);
    while (true) {
      const u64 least = lists[0][n - 1];  // 0: fewer threads than n have elements
      const float floor = value_of(static_cast<uint32_t>(least >> 32));
      if (tid == 0) s_found = 0;
      __syncthreads();
      int chunk = 0;
      for (int first = begin; first < end; first += kChunk, ++chunk) {
        if (least && chunk < kChunksKnown && chunk_tops[warp][chunk] < floor) continue;
        // Pieces that have one, then those one after another.
        unsigned has = 0;
#pragma unroll
        for (int j = 0; j < kScorePieces; ++j) {
          const int p = first + tid + j * kScoreThreads;
          if (p < end && !(least && E::largest(again(p)) < floor)) has |= 1u << j;
        }
        while (has) {
          const int p = first + tid + (__ffs(has) - 1) * kScoreThreads, at = row.first(p);
          has &= has - 1;
          float x[W];
          E::widen(again(p), x);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if ((least && x[i] < floor) || at + i < 0 || at + i >= V) continue;
            const u64 key = placed(x[i], at + i);
            if (key < least) continue;
            const int place = atomicAdd(&s_found, 1);
            if (place < kFound) found[place] = key;
          }
        }
      }
      __syncthreads();
      const int all = s_found, count = min(all, kFound);
      u64 list = 0;
      for (int i = 32 * warp; i < count; i += kScoreThreads) {
        const u64 more = warp_sort(i + lane < count ? found[i + lane] : 0, lane);
        list = i == 32 * warp ? more : warp_merge(list, more, lane);
      }
      lists[warp][lane] = list;
      merge_lists(lists, min(kScoreWarps, (count + 31) / 32), warp, lane);
      if (all <= kFound) break;
    }
  } else {
    __syncthreads();
  }
  // To the first CTA; the others are done then.
  cluster_wait();  // it has started
  if (warp == 0) {
    const Sums mine = sums_of_lanes(lane < kScoreWarps ? sums[lane] : Sums{-kInfinity, 0.0f, 0.0f, 0.0f}, 16);
    if (lane == 0) *of_rank(&ranks_sums[rank], 0) = mine;
  } else if (warp == 1 && n) {
    of_rank(&ranked[rank][0], 0)[lane] = lists[0][lane];
  }
  cluster_arrive();
  if (rank) return;
  cluster_wait();
  if (warp == 0) {
    const Sums all = sums_of_lanes(lane < ranks ? ranks_sums[lane] : Sums{-kInfinity, 0.0f, 0.0f, 0.0f}, kMaxCluster / 2);
    if (lane == 0) {
      // A row of nothing but -inf, with NaN or with +inf has no distribution.
      const bool none = !(fabsf(all.m) < kInfinity);
      const float nan = __int_as_float(0x7fffffff);
      const float log_z = none ? nan : log1pf(all.others + (all.equal - 1.0f));
      logprobs[r] = given ? (x_token - all.m) - log_z : nan;
      entropy[r] = log_z - all.weighted / (all.others + all.equal);
      s_log_z = log_z;
      s_m = all.m;
    }
  }
  if (n) {
    merge_lists(ranked, ranks, warp, lane);
    if (tid < n) {
      const u64 key = ranked[0][lane];
      const int64_t at = r * n + tid;
      top_ids[at] = place_of(key);
      top_logprobs[at] = (value_of(static_cast<uint32_t>(key >> 32)) - s_m) - s_log_z;
    }
  }
}

// ---- divergence ------------------------------------------------------------------------------------
// KL(P || Q) = E[d] + log E[e^-d] over P, d = a - b.  With any shift taken from d, t = d - shift,
// psi(t) = e^-t - 1 + t and x = E[psi] - E[t], it is
//   E[psi] + (log1p(x) - x),
// where nothing of first order in t is left to cancel: rows that hardly differ keep their digits in FP32.
// A shift is changed by D: psi(t + D) = e^-D psi(t) + psi(D) - (e^-D - 1) t.
// 1 + x = E[e^-t] is a difference, whose digits t must not be large for; rows of which it has too few left take another pass, with a
// sum of its own for it: E[t] + log E[e^-t].  (128 rows of 131072 FP32 99 us with the other pass, 30 without.)
constexpr int kComparePieces = 2;  // of a thread and row that are looked at together
constexpr int kCompareChunks = 2;  // that are on their way or looked at
constexpr int kCompareChunk = kComparePieces * kScoreThreads;
constexpr size_t kCompareRing = 2ull * kCompareChunks * kComparePieces * kScoreThreads * 16;  // of two rows
constexpr float kSlack = 2.0f;     // by which an a may be above its exponential's shift
constexpr float kNear = 60.0f;     // |t| and shifts of the single pass; beyond, and where a row has -inf alone, NaN or +inf, there is another

// psi(t) / t^2 for |t| up to 1/2: the series to t^6, whose last term the Chebyshev polynomial of degree six turns into
// lower ones; 3e-8 of the value.
__device__ __forceinline__ float psi_series(float t) {
  constexpr float last = 1.0f / 40320.0f;
  float p = -1.0f / 5040.0f;
  p = __fmaf_rn(p, t, 1.0f / 720.0f + 0.375f * last);
  p = __fmaf_rn(p, t, -1.0f / 120.0f);
  p = __fmaf_rn(p, t, 1.0f / 24.0f - 0.03515625f * last);
  p = __fmaf_rn(p, t, -1.0f / 6.0f);
  return __fmaf_rn(p, t, 0.5f + 0.00048828125f * last);
}
__device__ __forceinline__ float psi(float t) {
  return fabsf(t) <= 0.5f ? __fmul_rn(__fmul_rn(t, t), psi_series(t)) : (exp_fast(-t) - 1.0f) + t;
}

// Of some elements, with e = e^(a - m): sums of e, e t and e psi(t); whether the single pass does not hold for them.
struct Moments {
  float m, shift, mass, mean, rest;
  int beyond;
};

// What the single pass has of E[e^-t] = 1 + E[psi] - E[t], Q's part, times the mass: a difference.
__device__ __forceinline__ float other_of(const Moments& s) { return s.mass + (s.rest - s.mean); }
// Where it is small (Q is sure of a token, and t large for all others), its digits are lost: at 1/64 six bits of them.
constexpr float kLeastOther = 1.0f / 64.0f;
// A larger t makes e^-t smaller: of a large one the difference then keeps only what the digits have left, 2^-24 of it.
constexpr float kMostOther = 256.0f;

// The same of another shift of t.  mass, other: of all that are to be moved alike.
__device__ __forceinline__ void reshift(Moments& s, float shift, float mass, float other) {
  const float by = __fsub_rn(s.shift, shift);
  if (!(fabsf(by) <= kNear && (by >= 0.0f || other >= kLeastOther * mass) && (by <= 0.0f || other <= kMostOther * mass)))
    s.beyond = 1;
  const float more = psi(by), less = fabsf(by) <= 0.5f ? __fsub_rn(more, by) : exp_fast(-by) - 1.0f;  // e^-by - 1
  s.rest = s.rest + (less * (s.rest - s.mean) + more * s.mass);
  s.mean = __fmaf_rn(by, s.mass, s.mean);
  s.shift = shift;
}

// A warp's moments with the shifts m of the exponentials and `shift` of t, the same in all lanes.
__device__ __noinline__ Moments moved(Moments s, float m, float shift) {
  float mass = s.mass, other = other_of(s);  // the warp's
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    mass += __shfl_xor_sync(kFull, mass, w);
    other += __shfl_xor_sync(kFull, other, w);
  }
  reshift(s, shift, mass, other);
  const float f = exp_fast(__fsub_rn(s.m, m));
  s.mass *= f;
  s.mean *= f;
  s.rest *= f;
  return s;
}

// The lanes' moments as one, in every lane, with the shift of a lane that has the largest a: where nearly all of the
// mass is on one element, t is zero there, and the small parts of the others are not lost beside it.
__device__ __noinline__ Moments moments_of_lanes(Moments s) {
  float m = s.m;
#pragma unroll
  for (int w = 16; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, w));
  const bool has = s.mass > 0.0f;
  const unsigned having = __ballot_sync(kFull, has && s.m == m);
  const float shift = __shfl_sync(kFull, s.shift, having ? __ffs(having) - 1 : 0);
  if (has) reshift(s, shift, s.mass, other_of(s));
  const float f = has ? exp_fast(__fsub_rn(s.m, m)) : 0.0f;
  Moments all;
  all.m = m;
  all.shift = shift;
  all.mass = f * s.mass;
  all.mean = f * s.mean;
  all.rest = f * s.rest;
  all.beyond = s.beyond;
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    all.mass += __shfl_xor_sync(kFull, all.mass, w);
    all.mean += __shfl_xor_sync(kFull, all.mean, w);
    all.rest += __shfl_xor_sync(kFull, all.rest, w);
    all.beyond |= __shfl_xor_sync(kFull, all.beyond, w);
  }
  return all;
}

// What a CTA has of its row.
struct Compared {
  Moments moments;
  u64 tops[2];  // largest elements
};

// The largest elements of a thread's pieces of two rows' chunks of which `value` are the largest values, with their places;
// a chunk that starts at `end` has none.
template <typename T>
__device__ __noinline__ ulonglong2 largest_of_chunks(Row<T> a, Row<T> b, int2 first, int end, float2 value) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  uint4 v[2][kComparePieces];
#pragma unroll
  for (int j = 0; j < kComparePieces; ++j) {
    const int p = first.x + threadIdx.x + j * kScoreThreads, q = first.y + threadIdx.x + j * kScoreThreads;
    if (p < end) v[0][j] = a.load(p);
    if (q < end) v[1][j] = b.load(q);
  }
  int place[2] = {0x7fffffff, 0x7fffffff};
#pragma unroll
  for (int of = 0; of < 2; ++of)
#pragma unroll
    for (int j = 0; j < kComparePieces; ++j) {
      const int p = (of ? first.y : first.x) + threadIdx.x + j * kScoreThreads;
      if (p >= end) continue;
      float x[W];
      E::widen(v[of][j], x);
      const int at = a.first(p);
      const float most = of ? value.y : value.x;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if ((x[i] == most || (x[i] != x[i] && most != most)) && at + i >= 0 && at + i < a.columns) place[of] = min(place[of], at + i);
    }
  return make_ulonglong2(place[0] < 0x7fffffff ? placed(value.x, place[0]) : 0, place[1] < 0x7fffffff ? placed(value.y, place[1]) : 0);
}

// The single pass over a thread's pieces of a chunk whose exponentials' shift is larger than kScaled: a mask of a finite
// value, mostly.  `from`: its first slot.  Mass, mean, rest and the largest |t|.
template <typename T>
__device__ __noinline__ float4 large_moments(uint32_t ring, int from, float m, float shift) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int j = 0; j < kComparePieces; ++j) {
    float x[W], y[W];
    E::widen_bounded(load_shared16(ring_slot(ring, from + j)), x);
    E::widen_bounded(load_shared16(ring_slot(ring, from + kComparePieces + j)), y);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float e = exp_fast(__fsub_rn(x[i], m)), t = __fsub_rn(__fsub_rn(x[i], y[i]), shift);
      sum.x += e;
      sum.y = __fmaf_rn(e, t, sum.y);
      sum.z = __fmaf_rn(e, psi(t), sum.z);
      sum.w = fmaxf(sum.w, fabsf(t));
    }
  }
  return sum;
}

constexpr float kPart = 1.0f / 16.0f;
constexpr float kWeight = -745.0f;  // the logarithm of the least weight beside the largest, e^-745: what 64 bits hold
// Sums of the other pass: of e = e^(a - max a), of e t times kPart, of e psi(t) and of e^(b - b*), which is e e^-t and all of Q; whether
// Q has nothing where P has something.  In 64 bits, as a thread adds up to a thousand times.
struct FarMoments {
  double mass, mean, rest, other;
  int infinite;
};

// The other pass, over rows that are far apart or have -inf where the other has not.  What Q has where P has nothing adds
// to the rest as it is.
template <typename T>
__device__ __noinline__ FarMoments far_moments(Row<T> a, Row<T> b, int begin, int end, float most_a, float base_b) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  FarMoments sum = {0.0, 0.0, 0.0, 0.0, 0};
#pragma unroll 1
  for (int p = begin + threadIdx.x; p < end; p += kScoreThreads) {
    float x[W], y[W], mass = 0.0f, mean = 0.0f, rest = 0.0f, other = 0.0f;
    E::widen(a.load(p), x);
    E::widen(b.load(p), y);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      // Not (x - y) less a shift: where the rows are far apart, x - y has lost what x and y have beside that.  In
      // sixteenths, so that differences of the largest numbers and a piece's sum of them are finite.
      const float below = __fsub_rn(kPart * x[i], kPart * most_a), below_b = __fsub_rn(kPart * y[i], kPart * base_b);
      const float part = __fsub_rn(below, below_b), t = part / kPart, size = fabsf(t);
      const float e = exp_fast(below / kPart), of_b = exp_fast(below_b / kPart);
      const bool given = below >= kPart * kWeight;
      if (given && y[i] == -kInfinity) sum.infinite = 1;
      if (given && e == 0.0f) {  // t may be larger than e is small
        const double more = exp(static_cast<double>(below) / kPart) * part;
        sum.mean += more;
        sum.rest += more / kPart;
      }
      const float u = e > 0.0f ? __fmul_rn(e, t) : 0.0f;
      mass += e;
      mean += e > 0.0f ? __fmul_rn(e, part) : 0.0f;
      other += of_b;
      rest += size <= 16.0f ? __fmul_rn(e, psi(t)) : of_b - e + u;
    }
    sum.mass += mass;
    sum.mean += mean;
    sum.rest += rest;
    sum.other += other;
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    sum.mass += __shfl_xor_sync(kFull, sum.mass, w);
    sum.mean += __shfl_xor_sync(kFull, sum.mean, w);
    sum.rest += __shfl_xor_sync(kFull, sum.rest, w);
    sum.other += __shfl_xor_sync(kFull, sum.other, w);
    sum.infinite |= __shfl_xor_sync(kFull, sum.infinite, w);
  }
  return sum;
}

// One cluster per row; its CTAs share the row's pieces.  One pass over both rows: a warp takes its largest a so far
// as the exponentials' shift, and d at the largest a of its first elements as that of t.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, kScorePerSm)
    k_compare_logits(const void* reference, int64_t reference_stride, const void* logits, int64_t stride, int V,
                     float* divergence, uint8_t* agreement) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  extern __shared__ __align__(16) uint8_t compare_shared[];
  __shared__ Compared compared;
  __shared__ Moments moments[kScoreWarps];
  __shared__ FarMoments far[kScoreWarps];
  __shared__ u64 tops[2][kScoreWarps];
  __shared__ float highs[2][kScoreWarps];
  __shared__ int s_beyond;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = cluster_size(), rank = cluster_rank();
  const int64_t r = blockIdx.x / ranks;
  const uint32_t ring = shared_u32(compare_shared);
  grid_dependency_wait();
  grid_dependency_release();
  const Row<T> a(reference, reference_stride, r, V), b(logits, stride, r, V, a.shift);
  const int pieces = a.pieces();
  const int begin = static_cast<int>(static_cast<int64_t>(pieces) * rank / ranks);
  const int end = static_cast<int>(static_cast<int64_t>(pieces) * (rank + 1) / ranks);
  const int whole_from = a.whole(0) && b.whole(0) ? 0 : 1, whole_to = a.whole(pieces - 1) && b.whole(pieces - 1) ? pieces : pieces - 1;
  // Slots of a chunk: the pieces of a, then those of b.  -inf where there are no more.
  auto bring_chunk = [&](int first, int slot) {
    if (first >= whole_from && first + kCompareChunk <= min(end, whole_to) && b.aligned) {
      const T *x = a.data + a.first(first + tid), *y = b.data + b.first(first + tid);
#pragma unroll
      for (int j = 0; j < kComparePieces; ++j) {
        copy_async16(ring_slot(ring, slot + j), x + j * kScoreThreads * W);
        copy_async16(ring_slot(ring, slot + kComparePieces + j), y + j * kScoreThreads * W);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < kComparePieces; ++j) {
        const int p = first + tid + j * kScoreThreads;
        const uint4 none = make_uint4(E::kNone, E::kNone, E::kNone, E::kNone);
        store_shared16(ring_slot(ring, slot + j), p < end ? a.load(p) : none);
        store_shared16(ring_slot(ring, slot + kComparePieces + j), p < end ? b.load(p) : none);
      }
    }
    copy_async_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kCompareChunks; ++i) bring_chunk(begin + i * kCompareChunk, 2 * kComparePieces * i);

  float best_a = -kInfinity, best_b = -kInfinity;  // of the thread, NaN above all, and the first chunks that have them
  int chunk_a = begin, chunk_b = begin;
  Moments sum = {-kInfinity, 0.0f, 0.0f, 0.0f, 0.0f, 0};
  int slot = 0;
  for (int first = begin; first < end; first += kCompareChunk) {
    copy_async_wait<kCompareChunks - 1>();
    typename E::Top high_a = E::lowest(), high_b = E::lowest();
#pragma unroll
    for (int j = 0; j < kComparePieces; ++j) {
      E::fold(high_a, load_shared16(ring_slot(ring, slot + j)));
      E::fold(high_b, load_shared16(ring_slot(ring, slot + kComparePieces + j)));
    }
    const float top_a = E::value(high_a), top_b = E::value(high_b);
    if (!(top_a <= best_a) && best_a == best_a) {
      best_a = top_a;
      chunk_a = first;
    }
    if (!(top_b <= best_b) && best_b == best_b) {
      best_b = top_b;
      chunk_b = first;
    }
    const float chunk = warp_max_nan(top_a);
    // Too large to be scaled, or NaN.
    if (!(chunk <= kModerate) || top_b != top_b) sum.beyond = 1;
    if (chunk > sum.m + kSlack && fabsf(chunk) <= kModerate) {  // new shifts, the same in the whole warp: of its largest a
      float d = 0.0f;
      if (top_a == chunk) {
#pragma unroll 1
        for (int j = 0; j < kComparePieces; ++j) {
          float x[W], y[W];
          E::widen_bounded(load_shared16(ring_slot(ring, slot + j)), x);
          E::widen_bounded(load_shared16(ring_slot(ring, slot + kComparePieces + j)), y);
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (x[i] == chunk) d = __fsub_rn(x[i], y[i]);
        }
      }
      d = __shfl_sync(kFull, d, __ffs(__ballot_sync(kFull, top_a == chunk)) - 1);
      // Banned by b, or t would lose what x and y have beside the rows' distance.
      if (!(fabsf(d) <= kNear)) sum.beyond = 1;
      if (sum.m > -kInfinity) sum = moved(sum, chunk, d);
      sum.shift = d;
      sum.m = chunk;
    }
    if (!(fabsf(sum.m) <= kModerate)) {
      // P has had nothing yet: -inf, or a mask that leaves no weight beside any logit of moderate size.  If Q has ...
      if (!(top_b < -kModerate)) sum.beyond = 1;
    } else if (fabsf(sum.m) > kScaled) {
      const float4 more = large_moments<T>(ring, slot, sum.m, sum.shift);
      sum.mass += more.x;
      sum.mean += more.y;
      sum.rest += more.z;
      if (!(more.w <= kNear)) sum.beyond = 1;
    } else {
      const float m = sum.m, shift = sum.shift;
      const float c = __fmul_rn(m, kLog2E), back = exp2_fast(-__fmaf_rn(m, kLog2E, -c));
      const Pair scale = pair_of(kLog2E, kLog2E), base = pair_of(-c, -c), minus = pair_of(-1.0f, -1.0f), less = pair_of(-shift, -shift);
      Pair masses = pair_of(0.0f, 0.0f), means = masses, rests = masses;
      float widest = 0.0f;
#pragma unroll
      for (int j = 0; j < kComparePieces; ++j) {
        float x[W], y[W];
        E::widen_bounded(load_shared16(ring_slot(ring, slot + j)), x);
        E::widen_bounded(load_shared16(ring_slot(ring, slot + kComparePieces + j)), y);
        Pair t[W / 2];
        float wide = 0.0f;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          t[i] = pair_add(pair_fma(pair_of(y[2 * i], y[2 * i + 1]), minus, pair_of(x[2 * i], x[2 * i + 1])), less);
          float t0, t1;
          pair_split(t[i], t0, t1);
          wide = fmaxf(wide, fmaxf(fabsf(t0), fabsf(t1)));
        }
        widest = fmaxf(widest, wide);
        const bool small = wide <= 0.5f;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          float p0, p1, t0, t1;
          pair_split(pair_fma(pair_of(x[2 * i], x[2 * i + 1]), scale, base), p0, p1);
          pair_split(t[i], t0, t1);
          const Pair e = pair_of(exp2_fast(p0), exp2_fast(p1));
          masses = pair_add(masses, e);
          means = pair_fma(e, t[i], means);
          Pair value = pair_mul(pair_mul(t[i], t[i]), pair_of(psi_series(t0), psi_series(t1)));
          if (!small) {
            float v0, v1;
            pair_split(value, v0, v1);
            value = pair_of(fabsf(t0) <= 0.5f ? v0 : (exp_fast(-t0) - 1.0f) + t0,
                            fabsf(t1) <= 0.5f ? v1 : (exp_fast(-t1) - 1.0f) + t1);
          }
          rests = pair_fma(e, value, rests);
        }
      }
      if (!(widest <= kNear)) sum.beyond = 1;
      float s0, s1;
      pair_split(masses, s0, s1);
      sum.mass = __fmaf_rn(s0 + s1, back, sum.mass);
      pair_split(means, s0, s1);
      sum.mean = __fmaf_rn(s0 + s1, back, sum.mean);
      pair_split(rests, s0, s1);
      sum.rest = __fmaf_rn(s0 + s1, back, sum.rest);
    }
    bring_chunk(first + kCompareChunks * kCompareChunk, slot);
    slot += 2 * kComparePieces;
    if (slot == 2 * kComparePieces * kCompareChunks) slot = 0;
  }
  // The warps', the CTA's.
  const float high_a = warp_max_nan(best_a), high_b = warp_max_nan(best_b);
  {
    Moments all = sum;  // the shifts are the warp's
#pragma unroll
    for (int w = 16; w; w >>= 1) {
      all.mass += __shfl_xor_sync(kFull, all.mass, w);
      all.mean += __shfl_xor_sync(kFull, all.mean, w);
      all.rest += __shfl_xor_sync(kFull, all.rest, w);
      all.beyond |= __shfl_xor_sync(kFull, all.beyond, w);
    }
    if (lane == 0) {
      moments[warp] = all;
      highs[0][warp] = high_a;
      highs[1][warp] = high_b;
      tops[0][warp] = tops[1][warp] = 0;
    }
  }
  __syncthreads();
  {
    // The threads that have a largest value look for its place.
    float most_a = highs[0][lane % kScoreWarps], most_b = highs[1][lane % kScoreWarps];
    most_a = warp_max_nan(most_a);
    most_b = warp_max_nan(most_b);
    const bool has_a = best_a == most_a || (best_a != best_a && most_a != most_a);
    const bool has_b = best_b == most_b || (best_b != best_b && most_b != most_b);
    if (__any_sync(kFull, has_a || has_b)) {
      const ulonglong2 found = largest_of_chunks(a, b, make_int2(has_a ? chunk_a : end, has_b ? chunk_b : end), end, make_float2(best_a, best_b));
      const u64 top_a = warp_max(found.x), top_b = warp_max(found.y);
      if (lane == 0) {
        tops[0][warp] = top_a;
        tops[1][warp] = top_b;
      }
    }
  }
  if (warp == 0) {
    const Moments all = moments_of_lanes(lane < kScoreWarps ? moments[lane] : Moments{-kInfinity, 0.0f, 0.0f, 0.0f, 0.0f, 0});
    if (lane == 0) compared.moments = all;
  }
  __syncthreads();
  if (warp == 0) {
    const u64 top_a = warp_max(lane < kScoreWarps ? tops[0][lane] : 0), top_b = warp_max(lane < kScoreWarps ? tops[1][lane] : 0);
    if (lane == 0) {
      compared.tops[0] = top_a;
      compared.tops[1] = top_b;
    }
  }
  __syncthreads();
  cluster_meet();
  // The row's, in every CTA's first warp.
  Moments all = {};
  u64 top_a = 0, top_b = 0;
  if (warp == 0) {
    Compared of = {{-kInfinity, 0.0f, 0.0f, 0.0f, 0.0f, 0}, {0, 0}};
    if (lane < ranks) of = *of_rank(&compared, lane);
    all = moments_of_lanes(of.moments);
    top_a = warp_max(of.tops[0]);
    top_b = warp_max(of.tops[1]);
    if (lane == 0) {
      // Shifts that add up may have taken the sums beyond FP32.
      s_beyond = all.beyond || !(all.mass > 0.0f && fabsf(all.mean) < kInfinity && fabsf(all.rest) < kInfinity &&
                                 other_of(all) >= kLeastOther * all.mass);
      tops[0][0] = top_a;
      tops[1][0] = top_b;
    }
  }
  __syncthreads();
  double kl = 0.0;
  if (!s_beyond) {
    const double mean_of = static_cast<double>(all.mean) / all.mass, rest_of = static_cast<double>(all.rest) / all.mass;
    const double x = rest_of - mean_of;
    // The same number; where x is large, the two would only cancel each other.
    kl = fabs(x) < 0.5 ? rest_of + (log1p(x) - x) : mean_of + log1p(x);
  } else {
    const float most_a = value_of(static_cast<uint32_t>(tops[0][0] >> 32)), most_b = value_of(static_cast<uint32_t>(tops[1][0] >> 32));
    const float b_there = E::one(b.data + place_of(tops[0][0]));
    // Rows without a distribution (nothing but -inf, with NaN or with +inf); rows so far apart that e^(b - b*) overflows,
    // of which b's largest is b*.
    const bool none = !(fabsf(most_a) < kInfinity) || !(fabsf(most_b) < kInfinity), apart = !(most_b - b_there <= kNear);
    FarMoments mine = {};
    if (!none) mine = far_moments(a, b, begin, end, most_a, apart ? most_b : b_there);
    if (lane == 0) far[warp] = mine;
    __syncthreads();
    cluster_meet();
    if (rank == 0 && warp == 0) {
      FarMoments total = {};
      for (int i = 0; i < ranks * kScoreWarps; ++i) {
        const FarMoments of = *of_rank(&far[i % kScoreWarps], i / kScoreWarps);
        total.mass += of.mass;
        total.mean += of.mean;
        total.rest += of.rest;
        total.other += of.other;
        total.infinite |= of.infinite;
      }
      const double mean_of = total.mean / (kPart * total.mass), rest_of = total.rest / total.mass, x = rest_of - mean_of;
      if (none) {
        kl = __longlong_as_double(0x7fffffffffffffffll);
      } else if (total.infinite) {
        kl = kInfinity;
      } else {
        // E[|t|] is below E[psi] + 1: where that is large, 1 + x is lost in the difference, and has a sum of its own.
        kl = rest_of < 1.0 && fabs(x) < 0.5 ? rest_of + (log1p(x) - x) : mean_of + log(total.other / total.mass);
      }
    }
  }
  if (rank == 0 && tid == 0) {
    divergence[r] = static_cast<float>(kl < 0.0 ? 0.0 : kl);
    agreement[r] = place_of(top_a) == place_of(top_b);
  }
  cluster_meet();  // the others' shared memory has been read
}

// ---- host ------------------------------------------------------------------------------------------
constexpr int kMaxColumns = 1 << 21;

static int element_bytes(int type) { return type == CFM_TYPE_F32 ? 4 : 2; }

static int check_rows(const cfm_rows* rows, int most_columns) {
  if (!rows) return CFM_E_NULL;
  if (rows->type < CFM_TYPE_BF16 || rows->type > CFM_TYPE_F32) return CFM_E_UNSUPPORTED;
  if (rows->rows < 0 || rows->columns < 1 || rows->columns > most_columns) return CFM_E_SHAPE;
  if (rows->rows == 0) return 0;
  if (!rows->data) return CFM_E_NULL;
  if (rows->rows > 1 && rows->stride < rows->columns) return CFM_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(rows->data) % element_bytes(rows->type)) return CFM_E_SHAPE;
  return 0;
}

// CTAs that share a row: until the call has 256, more than one for most SMs, or a thread has one piece.  What a CTA does after its
// sums (5 to 8 us with top alternatives, all latency) grows with their number.  us of 1, 2, 4, 8 and 16 CTAs per row of 151936 BF16 logits,
// log probabilities: one row 14.5, 9.4, 6.9, 5.6, 4.0; 32 rows 14.8, 9.7, 8.1, 8.0, 8.5; 128 rows 15.8, 13.8, 15.2, 20.5, 24.5; 300 rows
// 34.7, 26.7, 30.2, 40.9, 53.6; 600 rows 43.0, 43.5, 53.6; 512 rows with 20 alternatives 63, 74, 102, 114.  Divergence: one row 32.7, 20.2,
// 14.0, 10.8, 9.4; 32 rows 34.4, 21.1, 16.1, 14.6, 21.6; 128 rows 35.4, 29.4, 31.0, 39.9, 63.1; 300 rows 83, 60, 64, 82; 600 rows 104, 99, 115.
// So from 256 to some 500 rows of such length two CTAs would be faster than the one taken; for short rows they are slower (300 rows of 8192:
// 6.2 and 8.1, 12.1 and 15.4; of 32003: 12.9 and 12.5, 30.7 and 29.7).
static int row_ranks(int rows, int columns, int type) {
  const int pieces = columns / (16 / element_bytes(type)) + 1;
  int ranks = 1;
  while (ranks < kMaxCluster && static_cast<int64_t>(rows) * ranks < 256 && pieces > ranks * kScoreThreads) ranks *= 2;
  return ranks;
}

template <typename T>
static int route(const cfm_rows* x, int K, int renormalize, void* ids, int ids64, void* weights, int weights16,
                 cudaStream_t stream) {
  const dim3 grid((x->rows + kRouteRows - 1) / kRouteRows), block(32 * kRouteRows);
  auto go = [&](auto kernel) {
    launch_dependent(kernel, grid, block, 0, stream, x->data, x->stride, x->rows, x->columns, K, renormalize, ids,
                     ids64, weights, weights16);
  };
  if (x->columns <= 64) go(k_route_tokens<T, 2>);
  else if (x->columns <= 128) go(k_route_tokens<T, 4>);
  else if (x->columns <= 256) go(k_route_tokens<T, 8>);
  else go(k_route_tokens<T, kRouteColumns / 32>);
  return launched();
}

template <typename T>
static int token_logprobs(const cfm_rows* x, const void* tokens, int tokens64, int n, float* logprobs, float* entropy,
                          int32_t* top_ids, float* top_logprobs, cudaStream_t stream) {
  const int ranks = row_ranks(x->rows, x->columns, x->type);
  if (const int code = allow_everything<k_token_logprobs<T>>(true)) return code;
  launch_clusters(k_token_logprobs<T>, dim3(x->rows * ranks), dim3(kScoreThreads), kRingBytes, ranks, stream, x->data,
                  x->stride, x->columns, tokens, tokens64, n, logprobs, entropy, top_ids, top_logprobs);
  return launched();
}

template <typename T>
static int compare_logits(const cfm_rows* a, const cfm_rows* b, float* divergence, uint8_t* agreement,
                          cudaStream_t stream) {
  const int ranks = row_ranks(a->rows, a->columns, a->type);
  if (const int code = allow_everything<k_compare_logits<T>>(true)) return code;
  launch_clusters(k_compare_logits<T>, dim3(a->rows * ranks), dim3(kScoreThreads), kCompareRing, ranks, stream, a->data,
                  a->stride, b->data, b->stride, a->columns, divergence, agreement);
  return launched();
}

}  // namespace cfm

using namespace cfm;

extern "C" {

int cfm_route_tokens(const cfm_rows* logits, int32_t top_k, int32_t renormalize, void* ids, int32_t ids_are_int64,
                     void* weights, int32_t weights_are_bf16, void* stream) {
  const int code = check_rows(logits, kRouteColumns);
  if (code) return code;
  if (top_k < 1 || top_k > 32 || top_k > logits->columns) return CFM_E_SHAPE;
  if (logits->rows == 0) return 0;
  if (!ids || !weights) return CFM_E_NULL;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (logits->type) {
    case CFM_TYPE_BF16: return route<__nv_bfloat16>(logits, top_k, renormalize, ids, ids_are_int64, weights, weights_are_bf16, s);
    case CFM_TYPE_F16: return route<__half>(logits, top_k, renormalize, ids, ids_are_int64, weights, weights_are_bf16, s);
    default: return route<float>(logits, top_k, renormalize, ids, ids_are_int64, weights, weights_are_bf16, s);
  }
}

int cfm_token_logprobs(const cfm_rows* logits, const void* tokens, int32_t tokens_are_int64, int32_t top,
                       float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, void* stream) {
  const int code = check_rows(logits, kMaxColumns);
  if (code) return code;
  if (top < 0 || top > kMaxTop || top > logits->columns) return CFM_E_SHAPE;
  if (logits->rows == 0) return 0;
  if (!tokens || !logprobs || !entropy || (top && (!top_ids || !top_logprobs))) return CFM_E_NULL;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (logits->type) {
    case CFM_TYPE_BF16: return token_logprobs<__nv_bfloat16>(logits, tokens, tokens_are_int64, top, logprobs, entropy, top_ids, top_logprobs, s);
    case CFM_TYPE_F16: return token_logprobs<__half>(logits, tokens, tokens_are_int64, top, logprobs, entropy, top_ids, top_logprobs, s);
    default: return token_logprobs<float>(logits, tokens, tokens_are_int64, top, logprobs, entropy, top_ids, top_logprobs, s);
  }
}

int cfm_compare_logits(const cfm_rows* reference, const cfm_rows* logits, float* divergence, uint8_t* agreement,
                       void* stream) {
  int code = check_rows(reference, kMaxColumns);
  if (!code) code = check_rows(logits, kMaxColumns);
  if (code) return code;
  if (reference->rows != logits->rows || reference->columns != logits->columns || reference->type != logits->type)
    return CFM_E_SHAPE;
  if (logits->rows == 0) return 0;
  if (!divergence || !agreement) return CFM_E_NULL;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (logits->type) {
    case CFM_TYPE_BF16: return compare_logits<__nv_bfloat16>(reference, logits, divergence, agreement, s);
    case CFM_TYPE_F16: return compare_logits<__half>(reference, logits, divergence, agreement, s);
    default: return compare_logits<float>(reference, logits, divergence, agreement, s);
  }
}

}  // extern "C"
