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

// The warp's values in descending order.
__device__ __forceinline__ u64 warp_sort(u64 v, int lane) {
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
__device__ __forceinline__ u64 warp_merge(u64 a, u64 b, int lane) {
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
    const int at = first(piece);
    if (whole(piece)) return __ldg(reinterpret_cast<const uint4*>(data + at));
    union {
      T e[W];
      uint4 v;
    } u;
    T none;
    if constexpr (sizeof(T) == 4) none = -kInfinity;
    else if constexpr (std::is_same<T, __half>::value) none = __ushort_as_half(0xfc00);
    else none = __ushort_as_bfloat16(0xff80);
#pragma unroll
    for (int i = 0; i < W; ++i) u.e[i] = at + i >= 0 && at + i < columns ? data[at + i] : none;
    return u.v;
  }
  // The largest element of a piece of which `value` is the largest value, with its place.
  __device__ u64 find(int piece, float value) const {
    const uint32_t key = ordered(value);
    const int at = first(piece);
    for (int i = 0; i < W; ++i)
      if (at + i >= 0 && at + i < columns && ordered(Element<T>::one(data + at + i)) == key)
        return static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(at + i));
    return 0;
  }
};

// Largest value that a thread has seen, and the first piece that has it.
struct Best {
  float value = -kInfinity;
  int piece = -1;
  __device__ void see(float v, int p) {
    if (piece < 0 || (!(v <= value) && value == value)) {
      value = v;
      piece = p;
    }
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
constexpr int kScoreThreads = 512;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreAhead = 4;  // pieces of a thread that are on their way together
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;

// Sums over elements x with the largest m: e^(x - m) without the `equal` elements that are m, and
// e^(x - m) (x - m).  Without them the sum keeps its digits where one token has nearly all probability:
// its log probability is then -log1p of the others' sum.
struct Sums {
  float m, equal, others, weighted;
};

// Tops of all warps' descending lists of 32, in the warps' first list; all threads.
__device__ __forceinline__ void merge_lists(u64 (*lists)[32], int count, int warp, int lane) {
  for (int step = 1; step < count; step <<= 1) {
    __syncthreads();
    if (warp % (2 * step) == 0 && warp + step < count)
      lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + step][lane], lane);
  }
  __syncthreads();
}

// One cluster per row; its CTAs share the row's pieces.  One pass over the row gives the sums: per warp,
// with the warp's largest value so far as the shift.  The top alternatives take a second pass, from the
// caches: the n-th largest of the threads' own maxima is not above the n-th largest element, so few elements
// are as large; those are sorted.  At most n threads have an element that large, which bounds their number
// for every input.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, 2)
    k_token_logprobs(const void* logits, int64_t stride, int V, const void* tokens, int tokens64, int n,
                     float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  extern __shared__ u64 found[];
  __shared__ u64 lists[kScoreWarps][32];
  __shared__ Sums sums[kScoreWarps];
  __shared__ double s_log_z;
  __shared__ float s_m;
  __shared__ int s_found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = cluster_size(), rank = cluster_rank();
  const int64_t r = blockIdx.x / ranks;
  grid_dependency_wait();
  grid_dependency_release();
  const Row<T> row(logits, stride, r, V);
  const int pieces = row.pieces();
  const int begin = static_cast<int>(static_cast<int64_t>(pieces) * rank / ranks);
  const int end = static_cast<int>(static_cast<int64_t>(pieces) * (rank + 1) / ranks);

  Best best;
  float m = -kInfinity, equal = 0.0f, others = 0.0f, weighted = 0.0f;
  uint4 next[kScoreAhead];
#pragma unroll
  for (int j = 0; j < kScoreAhead; ++j) {
    const int p = begin + tid + j * kScoreThreads;
    if (p < end) next[j] = row.load(p);
  }
  for (int first = begin; first < end; first += kScoreAhead * kScoreThreads) {
    uint4 v[kScoreAhead];
    float top[kScoreAhead], chunk = -kInfinity;
#pragma unroll
    for (int j = 0; j < kScoreAhead; ++j) {
      v[j] = next[j];
      const int p = first + tid + j * kScoreThreads;
      top[j] = -kInfinity;
      if (p < end) {
        top[j] = E::largest(v[j]);
        best.see(top[j], p);
        chunk = max_nan(chunk, top[j]);
      }
      const int ahead = p + kScoreAhead * kScoreThreads;
      if (ahead < end) next[j] = row.load(ahead);
    }
    chunk = warp_max_nan(chunk);
    if (!(chunk <= m) && m == m) {  // a new shift, the same in the whole warp; NaN stays
      const float step = m - chunk, f = m == -kInfinity ? 0.0f : exp_fast(step);
      const float all = others + equal;
      weighted = m == -kInfinity ? 0.0f : f * (weighted + step * all);
      others = f * all;
      equal = 0.0f;
      m = chunk;
    }
    if (m == -kInfinity) continue;  // nothing but -inf so far
#pragma unroll
    for (int j = 0; j < kScoreAhead; ++j) {
      if (top[j] == -kInfinity) continue;
      float x[W];
      E::widen(v[j], x);
      if (top[j] == m) {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (x[i] == m) {
            equal += 1.0f;
            x[i] = -kInfinity;
          }
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float d = fmaxf(__fsub_rn(x[i], m), -1e30f);  // -inf: adds nothing
        const float e = exp_fast(d);
        others += e;
        weighted = __fmaf_rn(e, d, weighted);
      }
    }
  }
  // NaN does not reach the sums by fmaxf: the shift says so.
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    equal += __shfl_xor_sync(kFull, equal, w);
    others += __shfl_xor_sync(kFull, others, w);
    weighted += __shfl_xor_sync(kFull, weighted, w);
  }
  if (lane == 0) sums[warp] = {m, equal, others, weighted};

  if (n) {
    // The thread's largest element, NaN above all.
    u64 top = best.piece >= 0 ? row.find(best.piece, best.value) : 0;
    lists[warp][lane] = warp_sort(top, lane);
    if (tid == 0) s_found = 0;
    merge_lists(lists, kScoreWarps, warp, lane);
    const u64 least = lists[0][n - 1];  // 0: fewer threads than n have elements, all of them are taken
    const float floor = value_of(static_cast<uint32_t>(least >> 32));
    for (int p = begin + tid; p < end; p += kScoreThreads) {
      const uint4 v = row.load(p);
      if (least && E::largest(v) < floor) continue;
      float x[W];
      E::widen(v, x);
      const int at = row.first(p);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (at + i < 0 || at + i >= V) continue;
        const u64 key = placed(x[i], at + i);
        if (key >= least) found[atomicAdd(&s_found, 1)] = key;
      }
    }
    __syncthreads();
    const int count = s_found;
    u64 list = 0;
    for (int i = 32 * warp; i < count; i += kScoreThreads) {
      const u64 more = warp_sort(i + lane < count ? found[i + lane] : 0, lane);
      list = i == 32 * warp ? more : warp_merge(list, more, lane);
    }
    lists[warp][lane] = list;
    merge_lists(lists, kScoreWarps, warp, lane);
  }
  __syncthreads();
  cluster_meet();
  if (rank == 0) {
    if (warp == 0) {
      const int entries = ranks * kScoreWarps;
      float largest = -kInfinity;
      for (int i = lane; i < entries; i += 32)
        largest = max_nan(largest, of_rank(&sums[i % kScoreWarps], i / kScoreWarps)->m);
      largest = warp_max_nan(largest);
      double equals = 0.0, rest = 0.0, total = 0.0;
      for (int i = lane; i < entries; i += 32) {
        const Sums s = *of_rank(&sums[i % kScoreWarps], i / kScoreWarps);
        if (s.m == largest) {
          equals += s.equal;
          rest += s.others;
          total += s.weighted;
        } else if (s.m > -kInfinity) {
          const float step = s.m - largest, f = expf(step);
          rest += f * (s.others + s.equal);
          total += f * (s.weighted + step * (s.others + s.equal));
        }
      }
#pragma unroll
      for (int w = 16; w; w >>= 1) {
        equals += __shfl_xor_sync(kFull, equals, w);
        rest += __shfl_xor_sync(kFull, rest, w);
        total += __shfl_xor_sync(kFull, total, w);
      }
      if (lane == 0) {
        // A row of nothing but -inf, with NaN or with +inf has no distribution.
        const bool none = !(fabsf(largest) < kInfinity);
        const double nan = __longlong_as_double(0x7fffffffffffffffll);
        const double log_z = none ? nan : log1p(rest + (equals - 1.0));
        const int64_t token = tokens64 ? static_cast<const int64_t*>(tokens)[r] : static_cast<const int32_t*>(tokens)[r];
        const bool given = token >= 0 && token < V;
        const float x = given ? E::one(row.data + token) : 0.0f;
        logprobs[r] = static_cast<float>(given && !none ? static_cast<double>(x - largest) - log_z : nan);
        entropy[r] = static_cast<float>(none ? nan : log_z - total / (rest + equals));
        s_log_z = log_z;
        s_m = largest;
      }
    }
    if (n) {
      __syncthreads();
      if (warp < ranks && warp > 0) lists[warp][lane] = of_rank(&lists[0][0], warp)[lane];
      merge_lists(lists, ranks, warp, lane);
      if (tid < n) {
        const u64 key = lists[0][lane];
        const int64_t at = r * n + tid;
        top_ids[at] = place_of(key);
        top_logprobs[at] = static_cast<float>(static_cast<double>(value_of(static_cast<uint32_t>(key >> 32)) - s_m) - s_log_z);
      }
    }
  }
  cluster_meet();  // the others' shared memory has been read
}

// ---- divergence ------------------------------------------------------------------------------------
// (e^-t - 1 + t) / t^2 for |t| up to 1/2, from the series: the first term left out is 4e-8 of the sum.
__device__ __forceinline__ float remainder_series(float t) {
  float p = 1.0f / 40320.0f;
  p = __fmaf_rn(p, t, -1.0f / 5040.0f);
  p = __fmaf_rn(p, t, 1.0f / 720.0f);
  p = __fmaf_rn(p, t, -1.0f / 120.0f);
  p = __fmaf_rn(p, t, 1.0f / 24.0f);
  p = __fmaf_rn(p, t, -1.0f / 6.0f);
  return __fmaf_rn(p, t, 0.5f);
}

// Over a row, with e = e^(a - max a): sums of e, of e t and of e (e^-t - 1 + t); or, where the rows are far
// apart, of e, of e t and of e^(b - max b).
struct Moments {
  float mass, shift, remainder;
  int infinite;
};

// One cluster per row; its CTAs share the row's pieces.  KL(P || Q) = E[d] + log E[e^-d] over P, d = a - b.
// With any shift taken from d, t = d - shift, and x = E[e^-t - 1 + t] - E[t], it is
//   E[e^-t - 1 + t] + (log1p(x) - x),
// where nothing of first order in t is left to cancel: rows that hardly differ keep their digits in FP32.
// The shift is d at the largest a, so the row's maxima are found first; the second pass reads from the caches.
// An element of which P has nothing adds its e^(b - b*) there, for the sum of all of them is Q's.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, 2)
    k_compare_logits(const void* reference, int64_t reference_stride, const void* logits, int64_t stride, int V,
                     float* divergence, uint8_t* agreement) {
  using E = Element<T>;
  constexpr int W = E::kWidth;
  __shared__ u64 tops[2][kScoreWarps];
  __shared__ u64 s_top[2];
  __shared__ Moments moments[kScoreWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = cluster_size(), rank = cluster_rank();
  const int64_t r = blockIdx.x / ranks;
  grid_dependency_wait();
  grid_dependency_release();
  const Row<T> a(reference, reference_stride, r, V), b(logits, stride, r, V, a.shift);
  const int pieces = a.pieces();
  const int begin = static_cast<int>(static_cast<int64_t>(pieces) * rank / ranks);
  const int end = static_cast<int>(static_cast<int64_t>(pieces) * (rank + 1) / ranks);

  Best best_a, best_b;
#pragma unroll 4
  for (int p = begin + tid; p < end; p += kScoreThreads) {
    const uint4 va = a.load(p), vb = b.load(p);
    best_a.see(E::largest(va), p);
    best_b.see(E::largest(vb), p);
  }
  const u64 top_a = warp_max(best_a.piece >= 0 ? a.find(best_a.piece, best_a.value) : 0);
  const u64 top_b = warp_max(best_b.piece >= 0 ? b.find(best_b.piece, best_b.value) : 0);
  if (lane == 0) {
    tops[0][warp] = top_a;
    tops[1][warp] = top_b;
  }
  __syncthreads();
  cluster_meet();
  if (warp < 2) {
    u64 top = 0;
    for (int i = lane; i < ranks * kScoreWarps; i += 32)
      top = max(top, *of_rank(&tops[warp][i % kScoreWarps], i / kScoreWarps));
    top = warp_max(top);
    if (lane == 0) s_top[warp] = top;
  }
  __syncthreads();
  const float most_a = value_of(static_cast<uint32_t>(s_top[0] >> 32));
  const float most_b = value_of(static_cast<uint32_t>(s_top[1] >> 32));
  const float b_there = E::one(b.data + place_of(s_top[0]));
  // Rows without a distribution (nothing but -inf, with NaN or with +inf); rows so far apart that e^(b - b*) overflows.
  const bool none = !(fabsf(most_a) < kInfinity) || !(fabsf(most_b) < kInfinity);
  const bool far = !(most_b - b_there <= 60.0f);
  const float base_b = far ? most_b : b_there, shift = most_a - base_b;

  Moments sum = {0.0f, 0.0f, 0.0f, 0};
  if (!none) {
#pragma unroll 2
    for (int p = begin + tid; p < end; p += kScoreThreads) {
      float x[W], y[W], t[W], widest = 0.0f;
      E::widen(a.load(p), x);
      E::widen(b.load(p), y);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        t[i] = __fsub_rn(__fsub_rn(x[i], y[i]), shift);
        widest = max_nan(widest, fabsf(t[i]));
      }
      if (widest <= 0.5f && !far) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float e = exp_fast(__fsub_rn(x[i], most_a)), u = __fmul_rn(e, t[i]);
          sum.mass += e;
          sum.shift += u;
          sum.remainder = __fmaf_rn(__fmul_rn(u, t[i]), remainder_series(t[i]), sum.remainder);
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float e = x[i] > -kInfinity ? exp_fast(__fsub_rn(x[i], most_a)) : 0.0f;
        if (x[i] > -kInfinity && y[i] == -kInfinity) sum.infinite = 1;
        const float u = e > 0.0f ? __fmul_rn(e, t[i]) : 0.0f;
        const float of_b = exp_fast(__fsub_rn(y[i], base_b));
        float more = of_b;
        if (!far) {
          const float size = fabsf(t[i]);
          more = size <= 0.5f    ? __fmul_rn(__fmul_rn(u, t[i]), remainder_series(t[i]))
                 : size <= 16.0f ? __fmul_rn(e, exp_fast(-t[i]) - 1.0f + t[i])
                                 : of_b - e + u;
        }
        sum.mass += e;
        sum.shift += u;
        sum.remainder += more;
      }
    }
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    sum.mass += __shfl_xor_sync(kFull, sum.mass, w);
    sum.shift += __shfl_xor_sync(kFull, sum.shift, w);
    sum.remainder += __shfl_xor_sync(kFull, sum.remainder, w);
    sum.infinite |= __shfl_xor_sync(kFull, sum.infinite, w);
  }
  if (lane == 0) moments[warp] = sum;
  __syncthreads();
  cluster_meet();
  if (rank == 0 && warp == 0) {
    double mass = 0.0, mean = 0.0, rest = 0.0;
    int infinite = 0;
    for (int i = lane; i < ranks * kScoreWarps; i += 32) {
      const Moments other = *of_rank(&moments[i % kScoreWarps], i / kScoreWarps);
      mass += other.mass;
      mean += other.shift;
      rest += other.remainder;
      infinite |= other.infinite;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) {
      mass += __shfl_xor_sync(kFull, mass, w);
      mean += __shfl_xor_sync(kFull, mean, w);
      rest += __shfl_xor_sync(kFull, rest, w);
      infinite |= __shfl_xor_sync(kFull, infinite, w);
    }
    if (lane == 0) {
      double kl;
      if (none) {
        kl = __longlong_as_double(0x7fffffffffffffffll);
      } else if (infinite) {
        kl = kInfinity;
      } else if (far) {
        kl = mean / mass + log(rest / mass);
      } else {
        const double remainder = rest / mass, x = remainder - mean / mass;
        // The same number; where x is large, remainder and x would only cancel each other.
        kl = fabs(x) < 0.5 ? remainder + (log1p(x) - x) : mean / mass + log1p(x);
      }
      divergence[r] = static_cast<float>(kl < 0.0 ? 0.0 : kl);
      agreement[r] = place_of(s_top[0]) == place_of(s_top[1]);
    }
  }
  cluster_meet();  // the others' shared memory has been read
}

// ---- host ------------------------------------------------------------------------------------------
constexpr int kMaxColumns = 1 << 21;  // elements that a thread may have to keep, 32 times over, fit shared memory

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

// CTAs that share a row.
static int row_ranks(int rows, int columns, int type) {
  const int pieces = columns / (16 / element_bytes(type)) + 1;
  int ranks = 1;
  while (ranks < kMaxCluster && static_cast<int64_t>(rows) * ranks < 592 && pieces > ranks * kScoreThreads) ranks *= 2;
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
  constexpr int W = Element<T>::kWidth;
  const int ranks = row_ranks(x->rows, x->columns, x->type);
  // Pieces of a CTA, and elements of a thread, at most.
  const int pieces = ((x->columns + W - 1) / W + 1 + ranks - 1) / ranks;
  const size_t shared = sizeof(u64) * n * W * ((pieces + kScoreThreads - 1) / kScoreThreads);
  if (shared > 40 * 1024) {
    const cudaError_t code = cudaFuncSetAttribute(k_token_logprobs<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(shared));
    if (code != cudaSuccess) return static_cast<int>(code);
  }
  launch_clusters(k_token_logprobs<T>, dim3(x->rows * ranks), dim3(kScoreThreads), shared, ranks, stream, x->data,
                  x->stride, x->columns, tokens, tokens64, n, logprobs, entropy, top_ids, top_logprobs);
  return launched();
}

template <typename T>
static int compare_logits(const cfm_rows* a, const cfm_rows* b, float* divergence, uint8_t* agreement,
                          cudaStream_t stream) {
  const int ranks = row_ranks(a->rows, a->columns, a->type);
  launch_clusters(k_compare_logits<T>, dim3(a->rows * ranks), dim3(kScoreThreads), 0, ranks, stream, a->data,
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
