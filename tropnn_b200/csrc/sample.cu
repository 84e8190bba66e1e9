// Sampling a token from logits with temperature, top-k, top-p and min-p and a given uniform
// number a row.
//
// Tokens are ranked by (logit descending, index ascending). With z = (x - max) * (1 / T) and
// e = exp(z), a token weighs the whole number W = round(2^31 e): sums of weights are exact in
// 64-bit integers, so no order of summation, split or batch changes a token. What is left is a
// prefix of the ranking:
//   top-k: the first k; top-p: those whose weight before them, among the top-k, is below
//   p * (weight of the top-k); min-p: those with e >= min_p; the first one always.
// The token is the first in index order whose running sum of kept weights passes
// floor(u * total). 2^-31 of the likeliest token's weight is finer than the 2^-24 of u itself.
// Temperature <= 0 (or NaN) takes the first of the ranking. A row without a finite or +inf logit,
// or with a NaN, gives -1.
//
// A row belongs to a cluster of 1 to 8 CTAs. The end of the prefix is found without sorting: a
// histogram over 2048 bins of z (counts and weights) names the bin that holds it, further ones over the
// rank keys of that bin's tokens name the logit; how many tokens of that logit stay is arithmetic, and
// which ones a running count in index order, taken together with the final sums. Where a top-k leaves at
// most 256 tokens, they go to the cluster's first CTA, which does the rest. Passes after the first skip
// vectors whose largest logit lies below what they look for. Where all the rows' CTAs are on the GPU at
// once and a row has a top-k or a top-p, the slices stay in shared memory between the passes. Else a row
// is streamed and the maxima of batches of four vectors alone are kept: later passes read again, from L2
// as far as it goes, the batches that can hold what they look for.
//
// Bound by instructions and barriers before HBM: every token of a top-p costs a call of expf (the whole
// weights have to be those of the exponentials alone, so none is approximated) and two shared-memory
// atomics, and each search step two cluster barriers. Measured on logits of 131072 bf16: greedy 512 rows
// 24 us (5.5 TB/s); min-p .05 512 rows 40 us, .5 2048 rows 100 us (5.4 TB/s); no cut 512 rows 82 us;
// top-p .95 64 rows 51 us, .9 512 rows 238 us; top-k 50 256 rows 34 us; one row of 32000 f32 with top-k
// 50 and top-p .9 12.7 us.
#include <cooperative_groups.h>

#include "common.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;
constexpr int kDigitBits = 11;
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kFew = 256;
// W >= 1 needs z >= ln(0.5 / 2^31) = -22.18: the bins cover the tokens that weigh anything.
constexpr float kLowestZ = -22.25f;
constexpr float kBinScale = kBins / -kLowestZ;
constexpr int64_t kSliceShared = 64 * 1024 + 64;  // bytes of logits a CTA, two on an SM
constexpr int64_t kSliceMost = 168 * 1024;        // one CTA on an SM

struct SampleArgs {
  const void *logits;
  int64_t inner, outer_stride, inner_stride, vocab;
  const float *uniforms;
  const float *temperature, *top_p, *min_p;  // one a row, or NULL: the value beside it
  const void *top_k;
  int top_k_dtype;
  float temperature_value, top_p_value, min_p_value;
  int64_t top_k_value;
  int64_t *tokens;
  int slice_vecs;   // 16-byte vectors of a CTA's slice
  int maxima_rows;  // batches a thread whose maxima are kept; 0: none
  int maxima_offset;
  bool halves;  // how the histogram holds weights
};

// Larger for larger logits; -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) != 0u ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) != 0u ? 0x80000000u : 0xFFFFFFFFu));
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One row's distribution.
struct Scale {
  float best, inv_t, temperature;
  // The minimum makes z(best) = 0 of a NaN: of inf - inf, or of 0 times an infinite 1 / T.
  __device__ __forceinline__ float z(float x) const { return fminf((x - best) * inv_t, 0.f); }
  __device__ __forceinline__ static uint32_t weight(float e) { return __float2uint_rn(e * 2147483648.f); }
  // -z in steps of 1 / kBinScale, to the nearest: adding it to 2^23 leaves the number in the low bits.
  // kBins (and nothing above): weighs nothing.
  __device__ __forceinline__ static int bin(float z) {
    return __float_as_int(fminf(fmaf(z, -kBinScale, 8388608.f), 8388608.f + kBins)) - 0x4B000000;
  }
  // A logit that every x with z(x) >= z0 is above, and one that it is below, rounding included.
  __device__ __forceinline__ float below(float z0) const {
    const float d = z0 * temperature;
    return fminf(best + d - 1e-5f * (fabsf(best) + fabsf(d)), best);
  }
  __device__ __forceinline__ float above(float z0) const {
    const float d = z0 * temperature;
    return fminf(best + d + 1e-5f * (fabsf(best) + fabsf(d)), best);
  }
  __device__ __forceinline__ float bin_low(int b) const { return below(-(b + 1) / kBinScale); }
  __device__ __forceinline__ float bin_high(int b) const { return above(-(b - 1) / kBinScale); }
};

// What the cluster's first CTA tells the others to do next.
enum Command { kDone = 0, kRefine = 1, kFresh = 2, kFinish = 3 };
struct Order {
  int command;
  int bin;
  uint32_t key_low, key_high;  // kRefine: the keys in question; kDone: those of the cut's logit
  uint32_t ties;               // kDone: how many tokens of that logit stay
};

struct Shared {
  uint64_t warp_sum[kWarps], slot_sum[kWarps][32];
  uint32_t warp_count[kWarps], slot_ties[kWarps][32];
  uint64_t sums[kMaxCluster];
  uint32_t ties[kMaxCluster], tie_weight[kMaxCluster];
  float maxima[kMaxCluster];
  uint32_t first_index[kMaxCluster];
  Order order;
  uint32_t listed, tied;
  // the first CTA's search
  int found;
  uint32_t found_count, found_count_before;
  uint64_t found_before, found_weight;
};

struct Histogram {
  uint32_t count[kBins], low[kBins], high[kBins];
};
struct Few {  // over the first CTA's histogram
  uint64_t key[kFew];  // rank keys: logit, then index
  uint32_t weight[kFew];
};
static_assert(sizeof(Few) <= sizeof(Histogram), "the list lies over the histogram");

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  // Keys of different logits are at least this far apart (a 16-bit logit leaves low f32 bits empty).
  static constexpr uint32_t kKeyStep = std::is_same<T, float>::value ? 1u : std::is_same<T, __half>::value ? 1u << 13 : 1u << 16;
  __device__ __forceinline__ static void unpack(const uint4 &q, float (&v)[kN]) {
    if constexpr (std::is_same<T, float>::value) {
      v[0] = __uint_as_float(q.x);
      v[1] = __uint_as_float(q.y);
      v[2] = __uint_as_float(q.z);
      v[3] = __uint_as_float(q.w);
    } else {
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        } else {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  }
};
// The largest element of a vector; PROPAGATE: NaN if one is.
template <typename T, bool PROPAGATE>
__device__ __forceinline__ float vec_max(const uint4 &q) {
  if constexpr (std::is_same<T, float>::value) {
    const float a = __uint_as_float(q.x), b = __uint_as_float(q.y), c = __uint_as_float(q.z), d = __uint_as_float(q.w);
    if constexpr (PROPAGATE) return max_nan(max_nan(a, b), max_nan(c, d));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 a = *reinterpret_cast<const __half2 *>(&q.x), b = *reinterpret_cast<const __half2 *>(&q.y),
                  c = *reinterpret_cast<const __half2 *>(&q.z), d = *reinterpret_cast<const __half2 *>(&q.w);
    const __half2 m = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162 *>(&q.x), b = *reinterpret_cast<const __nv_bfloat162 *>(&q.y),
                         c = *reinterpret_cast<const __nv_bfloat162 *>(&q.z), d = *reinterpret_cast<const __nv_bfloat162 *>(&q.w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
    return max_nan(__low2float(m), __high2float(m));
  }
}
template <typename T>
__device__ __forceinline__ T lowest_logit();
template <>
__device__ __forceinline__ float lowest_logit<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ __half lowest_logit<__half>() { return __ushort_as_half(0xFC00); }
template <>
__device__ __forceinline__ __nv_bfloat16 lowest_logit<__nv_bfloat16>() { return __ushort_as_bfloat16(0xFF80); }

template <typename T>
__device__ __forceinline__ uint4 nothing_vec() {  // -inf throughout
  const uint32_t w = std::is_same<T, float>::value ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}

// Vector v of the row's 16-byte grid, which starts at or before the row: elements outside the row
// are -inf and never read.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T *grid, int64_t v, int64_t lead, int64_t end) {
  constexpr int kN = Vec<T>::kN;
  const int64_t p = v * kN;
  if (p >= lead && p + kN <= end) return __ldg(reinterpret_cast<const uint4 *>(grid + p));
  alignas(16) T e[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) e[i] = p + i >= lead && p + i < end ? grid[p + i] : lowest_logit<T>();
  return *reinterpret_cast<const uint4 *>(e);
}

// Split barrier of the cluster: no CTA touches another's shared memory before all have started.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync(int ranks) {
  if (ranks > 1) cg::this_cluster().sync();
  else __syncthreads();
}

template <typename T>
__device__ __forceinline__ float lowest_finite() {
  return std::is_same<T, float>::value ? -3.4028234663852886e38f : std::is_same<T, __half>::value ? -65504.f : -3.3895313892515355e38f;
}
// Which elements of a lane's four vectors lie in [lo, hi] (as T, the bounds widened to it): bit n for the
// n-th 32-bit word's (low) element, 16 + n for its high one. Never one that is -inf: those fill the
// vectors past the slice and outside the row, which are not to be read.
template <typename T, bool BELOW>
__device__ __forceinline__ uint32_t mask_of(const uint4 (&q)[4], float lo, float hi) {
  lo = fmaxf(lo, lowest_finite<T>());
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = 4 * i + k;
      if constexpr (std::is_same<T, float>::value) {
        const float f = __uint_as_float(w[k]);
        if (f >= lo && (!BELOW || f <= hi)) mask |= 1u << n;
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 f = *reinterpret_cast<const __half2 *>(&w[k]);
        uint32_t in = __hge2_mask(f, __half2half2(__float2half_rd(lo)));
        if (BELOW) in &= __hle2_mask(f, __half2half2(__float2half_ru(hi)));
        mask |= in & (0x00010001u << n);
      } else {
        const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162 *>(&w[k]);
        uint32_t in = __hge2_mask(f, __bfloat162bfloat162(__float2bfloat16_rd(lo)));
        if (BELOW) in &= __hle2_mask(f, __bfloat162bfloat162(__float2bfloat16_ru(hi)));
        mask |= in & (0x00010001u << n);
      }
    }
  }
  return mask;
}
// Element (vector of the four, position in it) of a mask's bit.
template <typename T>
__device__ __forceinline__ void place_of(int bit, int &vector, int &element) {
  const int n = bit & 15;
  vector = n >> 2;
  element = sizeof(T) == 4 ? n & 3 : 2 * (n & 3) + (bit >> 4);
}

// The sum over a warp, in every lane.
__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
  const uint32_t a = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v) & 0xFFFFu);
  const uint32_t b = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 16) & 0xFFFFu);
  const uint32_t c = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 32) & 0xFFFFu);
  const uint32_t d = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 48));
  return a + (uint64_t(b) << 16) + (uint64_t(c) << 32) + (uint64_t(d) << 48);
}

// Inclusive prefix sums of a count and a weight over the block's threads, and their totals.
__device__ __forceinline__ void block_scan(uint32_t &count, uint64_t &weight, uint32_t &all_count, uint64_t &all_weight,
                                           Shared &sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t c = __shfl_up_sync(0xffffffffu, count, o);
    const uint64_t w = __shfl_up_sync(0xffffffffu, weight, o);
    if (lane >= o) {
      count += c;
      weight += w;
    }
  }
  __syncthreads();
  if (lane == 31) {
    sh.warp_count[warp] = count;
    sh.warp_sum[warp] = weight;
  }
  __syncthreads();
  uint32_t c = sh.warp_count[lane % kWarps];
  uint64_t w = sh.warp_sum[lane % kWarps];
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const uint32_t cb = __shfl_up_sync(0xffffffffu, c, o, kWarps);
    const uint64_t wb = __shfl_up_sync(0xffffffffu, w, o, kWarps);
    if ((lane % kWarps) >= o) {
      c += cb;
      w += wb;
    }
  }
  all_count = __shfl_sync(0xffffffffu, c, kWarps - 1);
  all_weight = __shfl_sync(0xffffffffu, w, kWarps - 1);
  const uint32_t cb = __shfl_sync(0xffffffffu, c, warp == 0 ? 0 : warp - 1);
  const uint64_t wb = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
  if (warp > 0) {
    count += cb;
    weight += wb;
  }
}

// SEARCH: some row may have a top-k or a top-p. Then with RESIDENT the slice stays in shared memory, else
// every pass reads global memory (L2) again. Without a search half as many threads a CTA stream the
// slice, RESIDENT false.
template <bool SEARCH>
constexpr int kBlock = SEARCH ? kThreads : kThreads / 2;
template <typename T, bool RESIDENT, bool SEARCH>
__global__ void __launch_bounds__(kBlock<SEARCH>, SEARCH ? 2 : 4) sample_kernel(const SampleArgs g) {
  constexpr int kThreads = kBlock<SEARCH>, kWarps = kThreads / 32;
  constexpr int kN = Vec<T>::kN;
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  Histogram &hist = *reinterpret_cast<Histogram *>(dynamic);
  Few &few = *reinterpret_cast<Few *>(dynamic);
  uint4 *kept_slice = reinterpret_cast<uint4 *>(dynamic + (SEARCH ? sizeof(Histogram) : 0));

  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const uint32_t row = blockIdx.x / static_cast<uint32_t>(ranks);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t outer = g.inner == 1 ? row : row / static_cast<uint32_t>(g.inner);  // both below 2^31
  const T *x = static_cast<const T *>(g.logits) + outer * g.outer_stride + (row - outer * g.inner) * g.inner_stride;
  const int64_t lead = static_cast<int64_t>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)), end = lead + g.vocab;
  const T *grid = x - lead;
  const int64_t vec0 = int64_t(rank) * g.slice_vecs;
  const int vecs = static_cast<int>(min64(g.slice_vecs, max(int64_t(0), (end + kN - 1) / kN - vec0)));
  auto element = [&](int v, int j) -> float {
    if constexpr (RESIDENT) return to_f32<T>(reinterpret_cast<const T *>(kept_slice)[v * kN + j]);
    else return ldg_f32(grid + (vec0 + v) * kN + j);
  };
  auto index0 = [&](int v) -> uint32_t { return static_cast<uint32_t>((vec0 + v) * kN - lead); };  // may wrap: unused then

  const float temperature = g.temperature != nullptr ? g.temperature[row] : g.temperature_value;
  float top_p = g.top_p != nullptr ? g.top_p[row] : g.top_p_value;
  float min_p = g.min_p != nullptr ? g.min_p[row] : g.min_p_value;
  int64_t top_k = g.top_k_value;
  if (g.top_k != nullptr)
    top_k = g.top_k_dtype == TROPNN_B200_I64 ? static_cast<const int64_t *>(g.top_k)[row] : static_cast<const int32_t *>(g.top_k)[row];
  // No token reaches a min-p above 1 (or NaN): the first one alone, as a top-p of 0 leaves it.
  if (!(min_p <= 1.f)) top_p = min_p = 0.f;
  const bool by_count = SEARCH && top_k > 0 && top_k < g.vocab;
  const bool by_weight = SEARCH && !(top_p >= 1.f);
  if (ranks > 1) cluster_arrive();

  // The slice, and the row's maximum (NaN where a logit is). Each warp has a stretch of the slice.
  const int per_warp = (vecs + kThreads - 1) / kThreads * 32;
  const int begin = min(warp * per_warp, vecs), stop = min(begin + per_warp, vecs);
  float m = -INFINITY;
  constexpr int kAhead = 4;
  const int batches = (stop - begin + 32 * kAhead - 1) / (32 * kAhead);  // of the warp
  // The batches' maxima, [batch][thread], where there is room for them.
  float *maxima = reinterpret_cast<float *>(dynamic + g.maxima_offset) + tid;
  const bool has_maxima = g.maxima_rows > 0;
  auto load4 = [&](int v, uint4 (&q)[kAhead]) {  // v and every 32nd vector after it, -inf past the stretch
    const int64_t p = (vec0 + v) * kN;
    if (p >= lead && v + 32 * (kAhead - 1) < stop && p + (32 * (kAhead - 1) + 1) * kN <= end) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) q[i] = __ldg(reinterpret_cast<const uint4 *>(grid + p) + 32 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        q[i] = nothing_vec<T>();
        if (v + 32 * i < stop) q[i] = load_vec<T>(grid, vec0 + v + 32 * i, lead, end);
      }
    }
  };
  auto again4 = [&](int v, uint4 (&q)[kAhead]) {  // the same in later passes
    if constexpr (RESIDENT) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        q[i] = nothing_vec<T>();
        if (v + 32 * i < stop) q[i] = kept_slice[v + 32 * i];
      }
    } else {
      load4(v, q);
    }
  };
  // Calls visit(x, index) for the logits of the warp's stretch that `mask` (of a batch) has a bit for,
  // with all lanes together: lanes without one bring -inf.
  auto each = [&](int v, uint32_t mask, auto visit) {
    while (__any_sync(0xffffffffu, mask != 0)) {
      float x = -INFINITY;
      uint32_t i = 0;
      if (mask != 0) {
        int vector, j;
        place_of<T>(__ffs(mask) - 1, vector, j);
        mask &= mask - 1;
        x = element(v + 32 * vector, j);
        i = index0(v + 32 * vector) + j;
      }
      visit(x, i);
    }
  };
  auto take = [&](int v, int n, const uint4 (&q)[kAhead]) {
    float batch = -INFINITY;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if constexpr (RESIDENT)
        if (v + 32 * i < stop) kept_slice[v + 32 * i] = q[i];
      batch = max_nan(batch, vec_max<T, true>(q[i]));
    }
    if (has_maxima) maxima[n * kThreads] = batch;
    m = max_nan(m, batch);
  };
  for (int v = begin + lane, n = 0; v < stop; v += 64 * kAhead, n += 2) {  // two batches on their way
    uint4 q[kAhead], r[kAhead];
    load4(v, q);
    load4(v + 32 * kAhead, r);
    take(v, n, q);
    if (v + 32 * kAhead < stop) take(v + 32 * kAhead, n + 1, r);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sh.warp_count[warp] = __float_as_uint(m);
  __syncthreads();
  if (ranks > 1) cluster_wait();
  if (warp == 0) {
    m = __uint_as_float(sh.warp_count[lane % kWarps]);
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane < ranks) *cluster.map_shared_rank(&sh.maxima[rank], lane) = m;
  }
  cluster_sync(ranks);
  Scale scale;
  scale.best = sh.maxima[0];
  for (int r = 1; r < ranks; ++r) scale.best = max_nan(scale.best, sh.maxima[r]);
  if (!(scale.best > -INFINITY)) {
    if (rank == 0 && tid == 0) g.tokens[row] = -1;
    return;
  }
  if (!(temperature > 0.f)) {
    uint32_t first = 0xFFFFFFFFu;
    for (int n = 0; n < batches; ++n) {
      const int v = begin + n * 32 * kAhead + lane;
      const bool some = v < stop && (!has_maxima || maxima[n * kThreads] >= scale.best);
      if (!__any_sync(0xffffffffu, some)) continue;
      uint4 q[kAhead];
      again4(some ? v : stop, q);
      each(v, mask_of<T, false>(q, scale.best, 0.f), [&](float x, uint32_t i) {
        if (x == scale.best) first = min(first, i);
      });
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.warp_count[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) first = min(first, sh.warp_count[w]);
      *cluster.map_shared_rank(&sh.first_index[rank], 0) = first;
    }
    cluster_sync(ranks);
    if (rank == 0 && tid == 0) {
      first = sh.first_index[0];
      for (int r = 1; r < ranks; ++r) first = min(first, sh.first_index[r]);
      g.tokens[row] = first;
    }
    return;
  }
  scale.temperature = temperature;
  scale.inv_t = fmaxf(1.f / temperature, __int_as_float(1));  // not 0 of an infinite T: -inf has to stay at -inf
  const float uniform = g.uniforms[row];
  auto target_of = [&](uint64_t total) -> uint64_t {
    const double place = floor(static_cast<double>(uniform) * static_cast<double>(total));
    const uint64_t target = place >= 1.0 ? static_cast<uint64_t>(place) : 0;
    return target > total - 1 ? total - 1 : target;
  };

  // Kept are the logits above cut_high and the first `ties` from cut_low to it (one value).
  float cut_low = -INFINITY, cut_high = -INFINITY;
  uint32_t ties = 0;
  if constexpr (SEARCH) if (by_count || by_weight) {
    // State of the first CTA's search: for the top-k's end, then for the top-p's.
    bool counting = by_count;
    const uint64_t limit_count = by_count ? static_cast<uint64_t>(top_k) : 0;
    double limit_weight = -1.0;  // not known yet
    auto limit_of = [&](uint64_t all) { return fmax(static_cast<double>(top_p) * static_cast<double>(all), 0.5); };
    uint64_t base_count = 0, base_weight = 0;  // before the keys in question
    // Of a top-k, nothing below the k-th largest of this slice's batch maxima: k tokens are above.
    float floor_x = scale.below(kLowestZ);
    bool few_above = false;
    if (by_count && has_maxima && g.maxima_rows >= 2) {
      for (int i = tid; i < kBins; i += kThreads) hist.count[i] = 0;
      if (tid == 0) sh.found = -1;
      __syncthreads();
      for (int n = 0; n < batches; ++n) {
        if (begin + n * 32 * kAhead + lane < stop) {
          const int b = Scale::bin(scale.z(maxima[n * kThreads]));
          if (b < kBins) atomicAdd(&hist.count[b], 1u);
        }
      }
      __syncthreads();
      const uint4 c = reinterpret_cast<const uint4 *>(hist.count)[tid];
      uint32_t upto = c.x + c.y + c.z + c.w, all;
      uint64_t none = 0, all_none;
      const uint32_t own = upto;
      block_scan(upto, none, all, all_none, sh);
      if (upto >= limit_count && upto - own < limit_count) sh.found = tid * 4 + 3;  // within four bins
      __syncthreads();
      few_above = sh.found >= 0;
      if (few_above) floor_x = scale.bin_low(sh.found);
      __syncthreads();
    }
    Order o;
    o.command = kFresh;
    o.bin = 0;
    o.key_low = o.key_high = 0;
    for (;;) {
      // A histogram: of all tokens by z, or of one bin's, between two keys, by the rest of their keys.
      const bool fresh = o.command == kFresh;
      const uint32_t range = o.key_high - o.key_low;  // keys, less one
      const int shift = max(0, 32 - __clz(range) - kDigitBits);
      for (int i = tid; i < kBins; i += kThreads) hist.count[i] = hist.low[i] = hist.high[i] = 0;
      __syncthreads();
      // A weight in two words: its halves, where no more than 2^16 tokens are a CTA's, so that neither
      // sum passes 32 bits; else the sum's low word and its carries.
      auto add_weight = [&](int b, uint32_t w) {
        if (g.halves) {
          atomicAdd(&hist.low[b], w & 0xFFFFu);
          atomicAdd(&hist.high[b], w >> 16);
        } else {
          const uint32_t old = atomicAdd(&hist.low[b], w);
          if (old + w < old) atomicAdd(&hist.high[b], 1u);
        }
      };
      if (fresh) {
        auto enter = [&](float x) {
          const float z = scale.z(x);
          const int b = Scale::bin(z);
          if (by_weight) {
            const uint32_t w = Scale::weight(expf(z));
            if (b < kBins) {
              add_weight(b, w);
              if (by_count) atomicAdd(&hist.count[b], 1u);
            }
          } else if (b < kBins) {
            atomicAdd(&hist.count[b], 1u);
          }
        };
        if (few_above) {
          for (int n = 0; n < batches; ++n) {
            const int v = begin + n * 32 * kAhead + lane;
            const bool some = v < stop && maxima[n * kThreads] >= floor_x;
            if (!__any_sync(0xffffffffu, some)) continue;
            uint4 q[kAhead];
            again4(some ? v : stop, q);
            each(v, mask_of<T, false>(q, floor_x, 0.f), [&](float x, uint32_t) { enter(x); });
          }
        } else {
          for (int n = 0; n < batches; ++n) {
            uint4 q[kAhead];
            again4(begin + n * 32 * kAhead + lane, q);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              if (vec_max<T, false>(q[i]) < floor_x) continue;
              float f[kN];
              Vec<T>::unpack(q[i], f);
#pragma unroll
              for (int j = 0; j < kN; ++j) enter(f[j]);
            }
          }
        }
      } else {
        const float low = logit_of(o.key_low), high = logit_of(o.key_high);
        for (int v0 = begin; v0 < stop; v0 += 32 * kAhead) {
          uint4 q[kAhead];
          again4(v0 + lane, q);
          each(v0 + lane, mask_of<T, true>(q, low, high), [&](float x, uint32_t) {
            const uint32_t down = o.key_high - key_of(x);  // larger keys first
            const float z = scale.z(x);
            if (down <= range && Scale::bin(z) == o.bin) {
              if (by_weight) {
                add_weight(down >> shift, Scale::weight(expf(z)));
              }
              atomicAdd(&hist.count[down >> shift], 1u);
            }
          });
        }
      }
      cluster_sync(ranks);
      if (rank == 0) {
        // All CTAs' bins (four a thread), and where the running count or weight reaches the limit.
        static_assert(kBinsPerThread == 4, "a bin a component");
        uint32_t c[4] = {0, 0, 0, 0};
        uint64_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          if (r < ranks) {
            const Histogram *h = cluster.map_shared_rank(&hist, r);
            if (by_count || !fresh) {
              const uint4 hc = reinterpret_cast<const uint4 *>(h->count)[tid];
              c[0] += hc.x;
              c[1] += hc.y;
              c[2] += hc.z;
              c[3] += hc.w;
            }
            if (by_weight) {
              const uint4 hl = reinterpret_cast<const uint4 *>(h->low)[tid], hh = reinterpret_cast<const uint4 *>(h->high)[tid];
              const int up = g.halves ? 16 : 32;
              w[0] += (uint64_t(hh.x) << up) + hl.x;
              w[1] += (uint64_t(hh.y) << up) + hl.y;
              w[2] += (uint64_t(hh.z) << up) + hl.z;
              w[3] += (uint64_t(hh.w) << up) + hl.w;
            }
          }
        }
        const uint32_t cs = c[0] + c[1] + c[2] + c[3];
        const uint64_t ws = w[0] + w[1] + w[2] + w[3];
        uint32_t upto_c = cs, all_count;
        uint64_t upto_w = ws, all_weight;
        if (tid == 0) sh.found = -1;
        block_scan(upto_c, upto_w, all_count, all_weight, sh);
        if (fresh) {
          if (counting && all_count < limit_count) counting = false;  // all that weigh anything stay
          if (!counting && limit_weight < 0.0) limit_weight = limit_of(all_weight);
        }
        const bool searching = counting || by_weight;
        if (searching) {
          uint64_t before_c = base_count + (upto_c - cs), before_w = base_weight + (upto_w - ws);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool open = counting ? before_c < limit_count : static_cast<double>(before_w) < limit_weight;
            const bool shut = counting ? before_c + c[i] >= limit_count
                                       : !(static_cast<double>(before_w + w[i]) < limit_weight);
            if (open && shut) {  // one of all
              sh.found = tid * 4 + i;
              sh.found_count = c[i];
              sh.found_count_before = static_cast<uint32_t>(before_c);
              sh.found_before = before_w;
              sh.found_weight = w[i];
            }
            before_c += c[i];
            before_w += w[i];
          }
        }
        __syncthreads();
        const int f = sh.found;
        Order next = o;
        if (!searching || f < 0) {
          next.command = kDone;
          next.key_low = next.key_high = 0;
        } else {
          base_count = sh.found_count_before;
          base_weight = sh.found_before;
          if (fresh) {
            next.bin = f;
            next.command = counting && base_count + sh.found_count <= kFew ? kFinish : kRefine;
            next.key_high = key_of(scale.bin_high(f));
            next.key_low = key_of(scale.bin_low(f));
          } else {
            next.command = kRefine;
            next.key_high = o.key_high - (static_cast<uint32_t>(f) << shift);
            const uint32_t left = next.key_high - o.key_low, span = (1u << shift) - 1u;
            next.key_low = next.key_high - min(left, span);
            if (next.key_high - next.key_low < Vec<T>::kKeyStep) {
              // One logit: its tokens weigh the same, and the first of them in index order stay.
              const uint64_t weight = sh.found_weight / sh.found_count;
              uint64_t stay = 0;
              if (counting) {
                stay = limit_count - base_count;
              } else {
                const double more = (limit_weight - static_cast<double>(base_weight)) / fmax(static_cast<double>(weight), 1.0);
                stay = more > 2.0 ? static_cast<uint64_t>(more) - 1 : 0;
                while (stay < sh.found_count && static_cast<double>(base_weight + stay * weight) < limit_weight) ++stay;
                while (stay > 1 && !(static_cast<double>(base_weight + (stay - 1) * weight) < limit_weight)) --stay;
              }
              next.command = kDone;
              next.ties = static_cast<uint32_t>(stay);
              if (counting && by_weight) {
                // The top-k's weight sets the top-p's limit, searched from the first bin.
                limit_weight = limit_of(base_weight + stay * weight);
                counting = false;
                base_count = base_weight = 0;
                next.command = kFresh;
              }
            }
          }
        }
        if (tid < ranks) *cluster.map_shared_rank(&sh.order, tid) = next;
        if (tid == 0) sh.listed = 0;
      }
      cluster_sync(ranks);
      o = sh.order;
      if (o.command == kDone) break;
      if (o.command == kFinish) {
        Few *to = cluster.map_shared_rank(&few, 0);
        uint32_t *listed = cluster.map_shared_rank(&sh.listed, 0);
        const float low = scale.bin_low(o.bin);
        for (int v0 = begin; v0 < stop; v0 += 32 * kAhead) {
          uint4 q[kAhead];
          again4(v0 + lane, q);
          each(v0 + lane, mask_of<T, false>(q, low, 0.f), [&](float x, uint32_t i) {
            if (x == -INFINITY || Scale::bin(scale.z(x)) > o.bin) return;
            const uint32_t place = atomicAdd(listed, 1u);
            if (place < kFew) to->key[place] = (uint64_t(key_of(x)) << 32) | (0xFFFFFFFFu - i);
          });
        }
        cluster_sync(ranks);
        if (rank != 0) return;
        // All that can be kept is here: rank each of the few tokens, keep, draw.
        const int n = static_cast<int>(min(sh.listed, uint32_t(kFew)));
        uint64_t key = 0;
        float e = 0.f;
        uint32_t w = 0;
        if (tid < n) {
          key = few.key[tid];
          e = expf(scale.z(logit_of(static_cast<uint32_t>(key >> 32))));
          w = Scale::weight(e);
          few.weight[tid] = w;
        }
        __syncthreads();
        uint32_t place = 0;
        uint64_t before = 0;
        if (tid < n) {
          for (int i = 0; i < n; ++i) {
            const bool ahead = few.key[i] > key;
            place += ahead ? 1u : 0u;
            before += ahead ? few.weight[i] : 0u;
          }
        }
        const bool top = tid < n && place < limit_count;
        uint32_t scratch_c = 0, all_c;
        uint64_t scratch_w = top ? w : 0u, all;
        block_scan(scratch_c, scratch_w, all_c, all, sh);
        bool keep = top && (!by_weight || static_cast<double>(before) < limit_of(all)) && e >= min_p;
        keep |= tid < n && place == 0;
        w = keep ? w : 0u;
        if (tid < n) few.weight[tid] = w;
        scratch_w = w;
        block_scan(scratch_c, scratch_w, all_c, all, sh);
        if (keep) {
          const uint32_t low = static_cast<uint32_t>(key);  // larger for lower indices
          uint64_t upto = 0;
          for (int i = 0; i < n; ++i) upto += static_cast<uint32_t>(few.key[i]) >= low ? few.weight[i] : 0u;
          const uint64_t target = target_of(all);
          if (upto > target && upto - w <= target) g.tokens[row] = 0xFFFFFFFFu - low;  // one of all
        }
        return;
      }
    }
    if (o.key_high != 0) {
      cut_low = logit_of(o.key_low);
      cut_high = logit_of(o.key_high);
      ties = o.ties;
    }
  }

  // The kept weights above the cut, and the tokens at it, of each warp's stretch of the slice, of each
  // CTA, of the row.
  const bool cutting = SEARCH && cut_high > -INFINITY;
  const float floor_x = fmaxf(cut_low, scale.below(fmaxf(kLowestZ, logf(min_p) - 1e-3f)));
  auto kept = [&](const uint4 &q, uint32_t (&w)[kN], uint32_t &at_cut) {  // at_cut: a bit an element
    float f[kN];
    Vec<T>::unpack(q, f);
    at_cut = 0;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const float e = expf(scale.z(f[j]));
      const bool in = e >= min_p && (!cutting || f[j] >= cut_low);
      w[j] = in ? Scale::weight(e) : 0u;
      if (cutting) at_cut |= w[j] != 0 && f[j] <= cut_high ? 1u << j : 0u;
    }
  };
  // The sums are also kept for 32 slots of consecutive batches a warp, so that the token is found by them.
  uint64_t sum = 0;
  uint32_t tied = 0, tie_weight = 0;
  const int per_slot = (batches + 31) / 32;
  for (int slot = 0, n = 0; n < batches; ++slot) {
    uint64_t lane_sum = 0;
    uint32_t lane_tied = 0;
    for (const int last = min(n + per_slot, batches); n < last; ++n) {
      const int v = begin + n * 32 * kAhead + lane;
      uint4 q[kAhead];
      bool some = v < stop;
      if (has_maxima && some) some = maxima[n * kThreads] >= floor_x;
      if (!__any_sync(0xffffffffu, some)) continue;
      again4(some ? v : stop, q);
      const uint32_t mask = mask_of<T, false>(q, floor_x, 0.f);
      if (__reduce_max_sync(0xffffffffu, __popc(mask)) <= kN) {  // few: one at a time
        each(v, mask, [&](float x, uint32_t) {
          const float e = expf(scale.z(x));
          const uint32_t w = e >= min_p && (!cutting || x >= cut_low) ? Scale::weight(e) : 0u;
          if (cutting && w != 0 && x <= cut_high) {
            ++lane_tied;
            tie_weight = w;  // the same for all
          } else {
            lane_sum += w;
          }
        });
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          uint32_t w[kN], at_cut;
          kept(q[i], w, at_cut);
          if (at_cut != 0) {
            lane_tied += __popc(at_cut);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
              if ((at_cut >> j) & 1u) {
                tie_weight = w[j];
                w[j] = 0;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < kN; ++j) lane_sum += w[j];
        }
      }
    }
    lane_sum = warp_sum64(lane_sum);
    lane_tied = __reduce_add_sync(0xffffffffu, lane_tied);
    if (lane == 0) {
      sh.slot_sum[warp][slot] = lane_sum;
      sh.slot_ties[warp][slot] = lane_tied;
    }
    sum += lane_sum;
    tied += lane_tied;
  }
  tie_weight = __reduce_max_sync(0xffffffffu, tie_weight);
  __syncthreads();
  if (tid == 0) sh.tied = 0;
  if (lane == 0) {
    sh.warp_sum[warp] = sum;
    sh.warp_count[warp] = tied;
  }
  __syncthreads();
  if (lane == 0 && tie_weight != 0) atomicMax(&sh.tied, tie_weight);
  uint64_t all = sh.warp_sum[lane % kWarps], before = lane < warp ? all : 0;
  const uint32_t warp_ties = sh.warp_count[lane % kWarps];
  uint32_t ties_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_ties : 0u);
  const uint32_t all_ties = __reduce_add_sync(0xffffffffu, lane < kWarps ? warp_ties : 0u);
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  __syncthreads();
  if (tid < ranks) {
    *cluster.map_shared_rank(&sh.sums[rank], tid) = all;
    *cluster.map_shared_rank(&sh.ties[rank], tid) = all_ties;
    *cluster.map_shared_rank(&sh.tie_weight[rank], tid) = sh.tied;
  }
  cluster_sync(ranks);
  uint64_t total = 0;
  uint32_t ties_total = 0;
  tie_weight = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) {
      before += sh.sums[r];
      ties_before += sh.ties[r];
    }
    total += sh.sums[r];
    ties_total += sh.ties[r];
    tie_weight = max(tie_weight, sh.tie_weight[r]);
  }
  total += uint64_t(min(ties_total, ties)) * tie_weight;
  before += uint64_t(min(ties_before, ties)) * tie_weight;
  sum += uint64_t(min(ties_before + tied, ties) - min(ties_before, ties)) * tie_weight;
  const uint64_t target = target_of(total);
  if (target < before || target >= before + sum) return;  // one warp of the cluster goes on
  const int slots = (batches + per_slot - 1) / per_slot;
  uint64_t slot_sum = lane < slots ? sh.slot_sum[warp][lane] : 0;
  uint32_t slot_ties = lane < slots ? sh.slot_ties[warp][lane] : 0, upto_ties = slot_ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t below = __shfl_up_sync(0xffffffffu, upto_ties, o);
    if (lane >= o) upto_ties += below;
  }
  const uint32_t first_tie = ties_before + upto_ties - slot_ties;
  slot_sum += uint64_t(min(first_tie + slot_ties, ties) - min(first_tie, ties)) * tie_weight;
  uint64_t upto_sum = slot_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t below = __shfl_up_sync(0xffffffffu, upto_sum, o);
    if (lane >= o) upto_sum += below;
  }
  const int slot = __ffs(__ballot_sync(0xffffffffu, before + upto_sum > target)) - 1;
  before += __shfl_sync(0xffffffffu, upto_sum - slot_sum, slot);
  ties_before = __shfl_sync(0xffffffffu, first_tie, slot);
  for (int n = slot * per_slot; n < batches; ++n) {
    const int v0 = begin + n * 32 * kAhead + lane;
    uint4 q[kAhead];
    again4(v0, q);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      uint32_t w[kN], at_cut;
      kept(q[i], w, at_cut);
      uint32_t rank_in = __popc(at_cut);  // of the lane's first token at the cut
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t below = __shfl_up_sync(0xffffffffu, rank_in, o);
        if (lane >= o) rank_in += below;
      }
      const uint32_t passed = __shfl_sync(0xffffffffu, rank_in, 31);
      rank_in += ties_before - __popc(at_cut);
      uint64_t mine = 0;
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        if ((at_cut >> j) & 1u) {
          if (rank_in >= ties) w[j] = 0;
          ++rank_in;
        }
        mine += w[j];
      }
      ties_before += passed;
      uint64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + upto > target);
      if (past != 0) {
        if (lane == __ffs(past) - 1) {
          uint64_t run = before + upto - mine;
          int found = -1;
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            run += w[j];
            if (found < 0 && run > target) found = j;
          }
          g.tokens[row] = index0(v0 + 32 * i) + found;
        }
        return;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
}

template <typename T>
int launch_sample(const char *what, SampleArgs g, int64_t rows, cudaStream_t stream) {
  int sms = 0;
  TB_CHECK(sm100::sm_count(&sms));
  const bool search = g.top_k != nullptr || g.top_k_value > 0 || g.top_p != nullptr || g.top_p_value < 1.f || g.min_p != nullptr ||
                      !(g.min_p_value <= 1.f);
  const int64_t row_bytes = g.vocab * int64_t(sizeof(T)) + 32;
  // With a search: a row's slices in shared memory, the fewest CTAs a row that keep two of them on an SM
  // and more while SMs are idle, as long as all the rows' CTAs are there at once (clusters of four and
  // more leave some of an SM's places empty). Else, and without a search: streamed by as many CTAs a row
  // as are there at once. Measured (131072 bf16 logits; in shared memory, streamed): top-p .9 of 1 row 31
  // and 34 us, 32 rows 35 and 41, 74 rows, which are not there at once, 72 and 56, 512 rows 334 and 238;
  // top-k 50 of 32 rows 16 and 19, of 74 29 and 18, of 512 142 and 62.
  // Splitting further costs barriers and, of a top-k, finds a lower floor: 8 rows of 32000 with a top-p
  // take 21 us by 4 or 8 CTAs and 26 by one; with top-k 50 1 row of 32000 f32 13.9 by 8 and 12.7 by 4, 16
  // rows of 131072 16.8 by 8 and 15.1 by 4, and 1 row of those 14.6 by 4 and 13.1 by 8.
  const int64_t slots = (search ? 2 : 4) * sms;
  const bool counting = g.top_k != nullptr || g.top_k_value > 0;
  const int64_t idle = counting ? sms / 2 : sms, least = counting ? 32 * 1024 : 16 * 1024;
  auto at_once = [&](int r) { return rows * r <= (r <= 2 ? slots : slots * 7 / 8); };
  int ranks = 1;
  while (ranks < kMaxCluster && (row_bytes > ranks * kSliceShared || (rows * ranks * 2 <= idle && row_bytes > ranks * least)))
    ranks *= 2;
  const bool resident = search && at_once(ranks) && ceil_div(row_bytes, ranks) <= kSliceMost;
  if (!resident) {
    ranks = 1;
    while (ranks < kMaxCluster && at_once(ranks * 2) && row_bytes > ranks * least) ranks *= 2;
  }
  const int64_t vecs = row_bytes / 16;
  const int64_t slice = ceil_div(vecs, ranks);
  TB_REQUIRE(rows * ranks <= 0x7fffffffLL && slice <= 0x7fffffffLL, TROPNN_B200_ERR_INVALID, "%s: too many rows", what);
  g.slice_vecs = static_cast<int>(slice);
  g.halves = slice * (16 / int64_t(sizeof(T))) <= 65536;
  size_t smem = 16;
  if (search) smem += sizeof(Histogram);
  if (resident) smem += static_cast<size_t>(slice) * 16;
  const int threads = search ? kBlock<true> : kBlock<false>;
  const int64_t batches = ceil_div(ceil_div(slice, threads), 4), room = resident ? 8 * 1024 : search ? 64 * 1024 : 48 * 1024;
  g.maxima_rows = 0;
  g.maxima_offset = static_cast<int>(smem);
  if (batches * threads * 4 <= room) {
    g.maxima_rows = static_cast<int>(batches);
    smem += static_cast<size_t>(batches) * threads * 4;
  }
  const void *kernel = !search    ? reinterpret_cast<const void *>(sample_kernel<T, false, false>)
                       : resident ? reinterpret_cast<const void *>(sample_kernel<T, true, true>)
                                  : reinterpret_cast<const void *>(sample_kernel<T, false, true>);
  // The static part counts too: above 48 KB in all the kernel has to be told.
  TB_CHECK(ensure_dynamic_smem(kernel, std::max<size_t>(smem, 49 * 1024), what));
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  void *args[] = {&g};
  cudaLaunchKernelExC(&config, kernel, args);
  return check_launch(what);
}

}  // namespace
}  // namespace tropnn_b200

using namespace tropnn_b200;

extern "C" int tropnn_b200_sample_tokens(const void *logits, int dtype, int64_t rows, int64_t inner, int64_t outer_stride,
                                         int64_t inner_stride, int64_t vocab, const float *uniforms,
                                         const float *temperature, float temperature_value, const void *top_k,
                                         int top_k_dtype, int64_t top_k_value, const float *top_p, float top_p_value,
                                         const float *min_p, float min_p_value, int64_t *tokens, void *stream) {
  const char *what = "sample_tokens";
  TB_REQUIRE(is_float_dtype(dtype), TROPNN_B200_ERR_DTYPE, "%s: logits dtype %d is not f32/f16/bf16", what, dtype);
  TB_REQUIRE(top_k == nullptr || top_k_dtype == TROPNN_B200_I64 || top_k_dtype == TROPNN_B200_I32, TROPNN_B200_ERR_DTYPE,
             "%s: top_k dtype %d is not i32/i64", what, top_k_dtype);
  TB_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && vocab >= 1 && vocab <= 0x7fffffffLL && inner >= 1 && inner <= 0x7fffffffLL,
             TROPNN_B200_ERR_INVALID, "%s: bad sizes (rows %lld, vocab %lld)", what, (long long)rows, (long long)vocab);
  if (rows == 0) return clear_error();
  TB_REQUIRE(logits != nullptr && uniforms != nullptr && tokens != nullptr, TROPNN_B200_ERR_INVALID, "%s: null pointer", what);
  TB_CHECK(check_current_device());
  SampleArgs g{};
  g.logits = logits;
  g.inner = inner;
  g.outer_stride = outer_stride;
  g.inner_stride = inner_stride;
  g.vocab = vocab;
  g.uniforms = uniforms;
  g.temperature = temperature;
  g.temperature_value = temperature_value;
  g.top_k = top_k;
  g.top_k_dtype = top_k_dtype;
  g.top_k_value = top_k_value;
  g.top_p = top_p;
  g.top_p_value = top_p_value;
  g.min_p = min_p;
  g.min_p_value = min_p_value;
  g.tokens = tokens;
  if (dtype == TROPNN_B200_F32) TB_CHECK(launch_sample<float>(what, g, rows, as_stream(stream)));
  else if (dtype == TROPNN_B200_F16) TB_CHECK(launch_sample<__half>(what, g, rows, as_stream(stream)));
  else TB_CHECK(launch_sample<__nv_bfloat16>(what, g, rows, as_stream(stream)));
  return clear_error();
}
