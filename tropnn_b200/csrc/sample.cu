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
// A row belongs to a cluster of 1 to 8 CTAs, each of which keeps its slice of the logits in shared
// memory: HBM is read once. The end of the prefix is found without sorting the row: a histogram
// over 2048 bins of z (counts and weights) names the bin that holds it, the few tokens of that bin
// go to the cluster's first CTA, which sorts them. A bin of more than 2048 tokens (equal or nearly
// equal logits) is first refined by the bits of its tokens' rank keys, 11 at a time.
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
constexpr int kList = 2048;
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kFew = 256;
// W >= 1 needs z >= ln(0.5 / 2^31) = -22.18: the bins cover the tokens that weigh anything.
constexpr float kLowestZ = -22.25f;
constexpr float kBinScale = kBins / -kLowestZ;
constexpr int64_t kSliceShared = 64 * 1024 + 64;  // bytes of logits a CTA, two (without a search three) on an SM
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
  int slice_vecs;  // 16-byte vectors of a CTA's slice
};

__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 ranks as +0
  const uint32_t key = b ^ ((b >> 31) != 0u ? 0xFFFFFFFFu : 0x80000000u);
  return (uint64_t(key) << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(k ^ ((k >> 31) != 0u ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One row's distribution.
struct Scale {
  float best, inv_t, temperature;
  bool only_best;  // an infinite best logit, or 1 / T past f32: nothing else weighs anything
  __device__ __forceinline__ float z(float x) const { return (x - best) * inv_t; }
  __device__ __forceinline__ float e(float x) const {
    if (only_best) return x == best ? 1.f : 0.f;
    return expf(z(x));
  }
  __device__ __forceinline__ static uint32_t weight(float e) { return __float2uint_rn(e * 2147483648.f); }
  // kBins and above: weighs nothing.
  __device__ __forceinline__ int bin(float x) const {
    if (only_best) return x == best ? 0 : kBins;
    return static_cast<int>(fminf(z(x) * -kBinScale, float(kBins)));
  }
  // A logit that every x with z(x) >= z0 is above, rounding included.
  __device__ __forceinline__ float below(float z0) const {
    if (only_best) return best;
    const float d = z0 * temperature;
    return best + d - 1e-5f * (fabsf(best) + fabsf(d));
  }
};

// What the cluster's first CTA tells the others to do next.
enum Command { kDone = 0, kGather = 1, kRefine = 2, kFinish = 3 };
struct Order {
  int command;
  int bin;
  int shift;           // kGather, kRefine: tokens of the bin with (key >> shift) == prefix; 64: all of the bin
  uint64_t prefix;
  float cut_logit;     // kDone: kept are x > cut_logit, and x == cut_logit up to cut_index
  uint32_t cut_index;
};

struct Shared {
  uint64_t warp_sum[kWarps];
  uint64_t sums[kMaxCluster];
  float maxima[kMaxCluster];
  uint32_t first_index[kMaxCluster];
  uint32_t warp_count[kWarps];
  Order order;
  uint32_t listed;
  // the first CTA's search
  int found;
  uint32_t found_count, found_count_before;
  uint64_t found_before, found_upto;
};

struct Histogram {
  uint32_t count[kBins], low[kBins], high[kBins];
};
struct Merged {
  uint32_t count[kBins];
  uint64_t weight[kBins];
};
constexpr size_t kSearchBytes = sizeof(Histogram) + sizeof(Merged);
static_assert(sizeof(Histogram) >= kList * sizeof(uint64_t), "the list lies over the histogram");

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
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

// The first n entries of `list` (room for kList), largest first; zeros fill up the power of two.
__device__ __forceinline__ void sort_list(uint64_t *list, uint32_t n) {
  uint32_t size = 2;
  while (size < n) size <<= 1;
  for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
  __syncthreads();
  for (uint32_t span = 2; span <= size; span <<= 1) {
    for (uint32_t d = span >> 1; d > 0; d >>= 1) {
      for (uint32_t i = threadIdx.x; i < size / 2; i += kThreads) {
        const uint32_t lo = ((i & ~(d - 1)) << 1) | (i & (d - 1)), hi = lo + d;
        const uint64_t p = list[lo], q = list[hi];
        if ((p < q) == ((lo & span) == 0)) {
          list[lo] = q;
          list[hi] = p;
        }
      }
      // Up to d = 32 a warp's pairs stay within its own 64 entries.
      if (d > 32 || d == 1) __syncthreads();
      else __syncwarp();
    }
  }
}

// RESIDENT: the slice stays in shared memory; else every pass reads global memory (L2) again.
// SEARCH: some row may have a top-k or a top-p.
template <typename T, bool RESIDENT, bool SEARCH>
__global__ void __launch_bounds__(kThreads, SEARCH ? 2 : 3) sample_kernel(const SampleArgs g) {
  constexpr int kN = Vec<T>::kN;
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  Histogram &hist = *reinterpret_cast<Histogram *>(dynamic);
  uint64_t *list = reinterpret_cast<uint64_t *>(dynamic);
  Merged &merged = *reinterpret_cast<Merged *>(dynamic + sizeof(Histogram));
  uint4 *kept_slice = reinterpret_cast<uint4 *>(dynamic + (SEARCH ? kSearchBytes : 0));

  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T *x = static_cast<const T *>(g.logits) + (row / g.inner) * g.outer_stride + (row % g.inner) * g.inner_stride;
  const int64_t lead = static_cast<int64_t>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)), end = lead + g.vocab;
  const T *grid = x - lead;
  const int64_t vec0 = int64_t(rank) * g.slice_vecs;
  const int vecs = static_cast<int>(min64(g.slice_vecs, max(int64_t(0), (end + kN - 1) / kN - vec0)));
  auto at = [&](int v) -> uint4 {
    if constexpr (RESIDENT) return kept_slice[v];
    else return load_vec<T>(grid, vec0 + v, lead, end);
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

  // The slice, and the row's maximum (NaN where a logit is).
  float m = -INFINITY;
  constexpr int kAhead = SEARCH ? 8 : 4;
  for (int v0 = tid; v0 < vecs; v0 += kThreads * kAhead) {
    uint4 q[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (v0 + i * kThreads < vecs) q[i] = load_vec<T>(grid, vec0 + v0 + i * kThreads, lead, end);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (v0 + i * kThreads < vecs) {
        if constexpr (RESIDENT) kept_slice[v0 + i * kThreads] = q[i];
        m = max_nan(m, vec_max<T, true>(q[i]));
      }
    }
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
    for (int v = tid; v < vecs; v += kThreads) {
      const uint4 q = at(v);
      if (vec_max<T, false>(q) < scale.best) continue;
      float f[kN];
      Vec<T>::unpack(q, f);
#pragma unroll
      for (int j = kN - 1; j >= 0; --j)
        if (f[j] == scale.best) first = min(first, index0(v) + j);
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
  scale.inv_t = 1.f / temperature;
  scale.only_best = scale.best == INFINITY || scale.inv_t == INFINITY;
  const float uniform = g.uniforms[row];
  auto target_of = [&](uint64_t total) -> uint64_t {
    const double place = floor(static_cast<double>(uniform) * static_cast<double>(total));
    const uint64_t target = place >= 1.0 ? static_cast<uint64_t>(place) : 0;
    return target > total - 1 ? total - 1 : target;
  };

  float cut_logit = -INFINITY;
  uint32_t cut_index = 0xFFFFFFFFu;
  if constexpr (SEARCH) if (by_count || by_weight) {
    // State of the first CTA's search: for the top-k's end, then for the top-p's.
    bool counting = by_count;
    const uint64_t limit_count = by_count ? static_cast<uint64_t>(top_k) : 0;
    double limit_weight = -1.0;  // not known yet
    auto limit_of = [&](uint64_t all) { return fmax(static_cast<double>(top_p) * static_cast<double>(all), 0.5); };
    uint64_t cut = 0;  // rank key of the last kept token
    uint32_t base_count = 0;
    uint64_t base_weight = 0;  // before the bin or digit in question
    int bin = -1, shift = 64;
    uint64_t prefix = 0;
    for (;;) {
      // A histogram: of all tokens by z (fresh), or of one bin's by the next bits of their keys.
      const bool fresh = bin < 0;
      for (int i = tid; i < kBins; i += kThreads) hist.count[i] = hist.low[i] = hist.high[i] = 0;
      __syncthreads();
      const int next_shift = shift == 64 ? 64 - kDigitBits : max(shift - kDigitBits, 0);
      const uint32_t digit_mask = (1u << ((shift == 64 ? 64 : shift) - next_shift)) - 1u;
      const float floor_x = scale.below(fresh ? kLowestZ : -(bin + 1) / kBinScale);
      for (int v = tid; v < vecs; v += kThreads) {
        const uint4 q = at(v);
        if (vec_max<T, false>(q) < floor_x) continue;
        float f[kN];
        Vec<T>::unpack(q, f);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          int b = scale.bin(f[j]);
          if (b >= kBins) continue;
          if (!fresh) {
            if (b != bin) continue;
            const uint64_t key = rank_key(f[j], index0(v) + j);
            if (shift < 64 && (key >> shift) != prefix) continue;
            b = kBins - 1 - static_cast<int>(static_cast<uint32_t>(key >> next_shift) & digit_mask);  // larger keys first
          }
          if (by_count) atomicAdd(&hist.count[b], 1u);
          if (by_weight) {
            const uint32_t w = Scale::weight(scale.e(f[j]));
            const uint32_t old = atomicAdd(&hist.low[b], w);
            if (old + w < old) atomicAdd(&hist.high[b], 1u);
          }
        }
      }
      cluster_sync(ranks);
      for (int i = rank * kThreads + tid; i < kBins; i += ranks * kThreads) {
        uint32_t c = 0;
        uint64_t w = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          if (r < ranks) {
            const Histogram *h = cluster.map_shared_rank(&hist, r);
            c += h->count[i];
            w += (uint64_t(h->high[i]) << 32) + h->low[i];
          }
        }
        Merged *to = cluster.map_shared_rank(&merged, 0);
        to->count[i] = c;
        to->weight[i] = w;
      }
      cluster_sync(ranks);
      bool listing = false;  // the first CTA has the bin's tokens
      Order o;
      do {
        if (rank == 0) {
          o.command = kDone;
          bool again;
          do {
            again = false;
            const uint32_t n = listing ? sh.listed : 0;
            if (n > kList) {  // known by its weight alone, the bin held too many
              o.command = kRefine;
              break;
            }
            if (listing) sort_list(list, n);
            // The place where the running count or weight reaches the limit: a bin, or a token.
            uint32_t c[kBinsPerThread], cs = 0;
            uint64_t w[kBinsPerThread], ws = 0;
#pragma unroll
            for (int i = 0; i < kBinsPerThread; ++i) {
              const uint32_t k = tid * kBinsPerThread + i;
              if (listing) {
                c[i] = k < n ? 1u : 0u;
                w[i] = k < n ? Scale::weight(scale.e(logit_of(list[k]))) : 0u;
              } else {
                c[i] = merged.count[k];
                w[i] = merged.weight[k];
              }
              cs += c[i];
              ws += w[i];
            }
            uint32_t upto_c = cs, all_count;
            uint64_t upto_w = ws, all_weight;
            block_scan(upto_c, upto_w, all_count, all_weight, sh);
            if (fresh && !listing) {
              if (counting && all_count < limit_count) counting = false;  // all that weigh anything stay
              if (!counting && limit_weight < 0.0) limit_weight = limit_of(all_weight);
            }
            if (tid == 0) sh.found = -1;
            __syncthreads();
            const bool searching = counting || by_weight;
            if (searching) {
              uint64_t before_c = uint64_t(base_count) + (upto_c - cs), before_w = base_weight + (upto_w - ws);
#pragma unroll
              for (int i = 0; i < kBinsPerThread; ++i) {
                const bool open = counting ? before_c < limit_count : static_cast<double>(before_w) < limit_weight;
                const bool shut = counting ? before_c + c[i] >= limit_count
                                           : !(static_cast<double>(before_w + w[i]) < limit_weight);
                if (open && shut) {  // one of all
                  sh.found = tid * kBinsPerThread + i;
                  sh.found_count = c[i];
                  sh.found_count_before = static_cast<uint32_t>(before_c);
                  sh.found_before = before_w;
                  sh.found_upto = before_w + w[i];
                }
                before_c += c[i];
                before_w += w[i];
              }
            }
            __syncthreads();
            const int f = sh.found;
            if (!searching || f < 0) break;
            if (listing) {
              cut = list[f];
              if (counting && by_weight) {
                // The top-k ends here; its weight sets the top-p's limit, searched from the first bin.
                counting = false;
                limit_weight = limit_of(sh.found_upto);
                base_count = 0;
                base_weight = 0;
                bin = -1;
                shift = 64;
                if (fresh) again = true;  // the histogram of all tokens is still there
                else o.command = kRefine;
                listing = false;
              }
              __syncthreads();  // sh.found and the list have been read
              continue;
            }
            if (fresh && counting && sh.found_count_before + sh.found_count <= kFew) {
              bin = f;
              o.command = kFinish;
              break;
            }
            base_count = sh.found_count_before;
            base_weight = sh.found_before;
            if (fresh) {
              bin = f;
            } else {
              const int bits = (shift == 64 ? 64 : shift) - next_shift;
              prefix = (shift == 64 ? 0 : prefix << bits) | static_cast<uint64_t>(kBins - 1 - f);
              shift = next_shift;
            }
            o.command = by_count && sh.found_count > kList ? kRefine : kGather;
          } while (again);
          o.bin = bin;
          o.shift = shift;
          o.prefix = prefix;
          o.cut_logit = cut == 0 ? -INFINITY : logit_of(cut);
          o.cut_index = cut == 0 ? 0xFFFFFFFFu : index_of(cut);
          __syncthreads();
          if (tid < ranks) *cluster.map_shared_rank(&sh.order, tid) = o;
          if (tid == 0) sh.listed = 0;
        }
        cluster_sync(ranks);
        o = sh.order;
        bin = o.bin;
        shift = o.shift;
        prefix = o.prefix;
        listing = o.command == kGather || o.command == kFinish;
        if (listing) {
          uint32_t *listed = cluster.map_shared_rank(&sh.listed, 0);
          uint64_t *to = cluster.map_shared_rank(list, 0);
          const float floor_bin = scale.below(-(bin + 1) / kBinScale);
          for (int v = tid; v < vecs; v += kThreads) {
            const uint4 q = at(v);
            if (vec_max<T, false>(q) < floor_bin) continue;
            float f[kN];
            Vec<T>::unpack(q, f);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
              const int b = scale.bin(f[j]);
              if (o.command == kFinish ? b > bin : b != bin) continue;
              const uint64_t key = rank_key(f[j], index0(v) + j);
              if (shift < 64 && (key >> shift) != prefix) continue;
              const uint32_t place = atomicAdd(listed, 1u);
              if (place < kList) to[place] = key;
            }
          }
          cluster_sync(ranks);
          if (o.command == kFinish) {
            if (rank != 0) return;
            // All that can be kept is here: rank each of the few tokens, keep, draw.
            const int n = static_cast<int>(sh.listed);
            uint32_t *weights = merged.count;
            uint64_t key = 0;
            float e = 0.f;
            uint32_t w = 0;
            if (tid < n) {
              key = list[tid];
              e = scale.e(logit_of(key));
              w = Scale::weight(e);
              weights[tid] = w;
            }
            __syncthreads();
            uint32_t place = 0;
            uint64_t before = 0;
            if (tid < n) {
              for (int i = 0; i < n; ++i) {
                const bool ahead = list[i] > key;
                place += ahead ? 1u : 0u;
                before += ahead ? weights[i] : 0u;
              }
            }
            const bool top = tid < n && place < limit_count;
            uint32_t scratch_c = 0, all_c;
            uint64_t scratch_w = top ? w : 0u, all;
            block_scan(scratch_c, scratch_w, all_c, all, sh);
            bool keep = top && (!by_weight || static_cast<double>(before) < limit_of(all)) && e >= min_p;
            keep |= tid < n && place == 0;
            w = keep ? w : 0u;
            __syncthreads();
            if (tid < n) weights[tid] = w;
            scratch_w = w;
            block_scan(scratch_c, scratch_w, all_c, all, sh);
            if (keep) {
              const uint32_t index = index_of(key);
              uint64_t upto = 0;
              for (int i = 0; i < n; ++i) upto += index_of(list[i]) <= index ? weights[i] : 0u;
              const uint64_t target = target_of(all);
              if (upto > target && upto - w <= target) g.tokens[row] = index;  // one of all
            }
            return;
          }
        }
      } while (listing);
      if (o.command == kDone) {
        cut_logit = o.cut_logit;
        cut_index = o.cut_index;
        break;
      }
    }
  }

  // The kept weights of each warp's stretch of the slice, of each CTA, of the row.
  const bool cutting = cut_logit > -INFINITY;
  const float floor_x = fmaxf(cut_logit, scale.below(fmaxf(kLowestZ, logf(min_p) - 1e-3f)));
  auto kept = [&](const uint4 &q, int v, uint32_t (&w)[kN]) {
    float f[kN];
    Vec<T>::unpack(q, f);
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const float e = scale.e(f[j]);
      bool in = e >= min_p;
      if (SEARCH && cutting) in &= f[j] > cut_logit || (f[j] == cut_logit && index0(v) + j <= cut_index);
      w[j] = in ? Scale::weight(e) : 0u;
    }
  };
  const int per_warp = (vecs + kThreads - 1) / kThreads * 32;
  const int begin = min(warp * per_warp, vecs), stop = min(begin + per_warp, vecs);
  uint64_t sum = 0;
  for (int v = begin + lane; v < stop; v += 32) {
    const uint4 q = at(v);
    if (vec_max<T, false>(q) < floor_x) continue;
    uint32_t w[kN];
    kept(q, v, w);
#pragma unroll
    for (int j = 0; j < kN; ++j) sum += w[j];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) sh.warp_sum[warp] = sum;
  __syncthreads();
  uint64_t all = sh.warp_sum[lane % kWarps], before = lane < warp ? all : 0;
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (tid < ranks) *cluster.map_shared_rank(&sh.sums[rank], tid) = all;
  cluster_sync(ranks);
  uint64_t total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += sh.sums[r];
    total += sh.sums[r];
  }
  const uint64_t target = target_of(total);
  if (target < before || target >= before + sum) return;  // one warp of the cluster goes on
  for (int v0 = begin; v0 < stop; v0 += 32) {
    const int v = v0 + lane;
    uint32_t w[kN];
    uint64_t mine = 0;
    if (v < stop) {
      kept(at(v), v, w);
#pragma unroll
      for (int j = 0; j < kN; ++j) mine += w[j];
    }
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
        g.tokens[row] = index0(v) + found;
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <typename T>
int launch_sample(const char *what, SampleArgs g, int64_t rows, cudaStream_t stream) {
  int sms = 0;
  TB_CHECK(sm100::sm_count(&sms));
  // The fewest CTAs a row that keep its slices at two CTAs an SM, more while SMs are idle.
  const int64_t row_bytes = g.vocab * int64_t(sizeof(T)) + 32;
  int ranks = 1;
  while (ranks < kMaxCluster && (row_bytes > ranks * kSliceShared || (rows * ranks * 2 <= sms && row_bytes > ranks * 4096)))
    ranks *= 2;
  const int64_t vecs = row_bytes / 16;
  const int64_t slice = ceil_div(vecs, ranks);
  const bool resident = slice * 16 <= kSliceMost;
  const bool search = g.top_k != nullptr || g.top_k_value > 0 || g.top_p != nullptr || g.top_p_value < 1.f || g.min_p != nullptr ||
                      !(g.min_p_value <= 1.f);
  TB_REQUIRE(rows * ranks <= 0x7fffffffLL && slice <= 0x7fffffffLL, TROPNN_B200_ERR_INVALID, "%s: too many rows", what);
  g.slice_vecs = static_cast<int>(slice);
  const size_t smem = (search ? kSearchBytes : 0) + 16 + (resident ? static_cast<size_t>(slice) * 16 : 0);
  const void *kernel = resident ? (search ? reinterpret_cast<const void *>(sample_kernel<T, true, true>)
                                          : reinterpret_cast<const void *>(sample_kernel<T, true, false>))
                                : (search ? reinterpret_cast<const void *>(sample_kernel<T, false, true>)
                                          : reinterpret_cast<const void *>(sample_kernel<T, false, false>));
  TB_CHECK(ensure_dynamic_smem(kernel, smem, what));
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  config.blockDim = dim3(kThreads);
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
  TB_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && vocab >= 1 && vocab <= 0x7fffffffLL && inner >= 1,
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
