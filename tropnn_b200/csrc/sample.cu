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
// W >= 1 needs z >= ln(0.5 / 2^31) = -22.18: the bins cover the tokens that weigh anything.
constexpr float kBinScale = kBins / 22.25f;
constexpr int64_t kSliceTwoPerSm = 64 * 1024;  // bytes of logits a CTA, two CTAs on an SM
constexpr int64_t kSliceMost = 168 * 1024;     // one CTA on an SM

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
  float best, inv_t;
  bool only_best;  // an infinite best logit, or 1 / T past f32: nothing else weighs anything
  __device__ __forceinline__ float z(float x) const { return (x - best) * inv_t; }
  __device__ __forceinline__ float e(float x) const {
    if (only_best) return x == best ? 1.f : 0.f;
    return expf(z(x));
  }
  __device__ __forceinline__ static uint32_t weight(float e) { return __float2uint_rn(e * 2147483648.f); }
  __device__ __forceinline__ int bin(float x) const {
    if (only_best) return 0;  // only the tokens at best weigh anything
    return min(static_cast<int>(z(x) * -kBinScale), kBins - 1);
  }
};

// What the cluster's first CTA tells the others to do next.
enum Command { kDone = 0, kGather = 1, kRefine = 2 };
struct Order {
  int command;
  int bin;
  int shift;           // tokens of the bin with (key >> shift) == prefix; 64: all of the bin
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
  int found_bin;
  uint32_t found_count;
  uint64_t found_before;
  uint32_t found_count_before;
  uint64_t total;
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

// RESIDENT: the slice stays in shared memory; else every pass reads global memory (L2) again.
template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs g) {
  constexpr int kN = Vec<T>::kN;
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  Histogram &hist = *reinterpret_cast<Histogram *>(dynamic);
  uint64_t *list = reinterpret_cast<uint64_t *>(dynamic);
  Merged &merged = *reinterpret_cast<Merged *>(dynamic + sizeof(Histogram));
  uint4 *kept_slice = reinterpret_cast<uint4 *>(dynamic + kSearchBytes);

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
  if (!(min_p <= 1.f)) top_p = min_p = 0.f;  // no token reaches it: the first one alone
  int64_t top_k = g.top_k_value;
  if (g.top_k != nullptr)
    top_k = g.top_k_dtype == TROPNN_B200_I64 ? static_cast<const int64_t *>(g.top_k)[row] : static_cast<const int32_t *>(g.top_k)[row];
  const bool by_count = top_k > 0 && top_k < g.vocab;
  const bool by_weight = !(top_p >= 1.f);

  if (ranks > 1) cluster_arrive();

  // The slice, and the row's maximum (NaN where a logit is).
  float m = -INFINITY;
  constexpr int kAhead = 4;
  for (int v0 = tid; v0 < vecs; v0 += kThreads * kAhead) {
    uint4 q[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (v0 + i * kThreads < vecs) q[i] = load_vec<T>(grid, vec0 + v0 + i * kThreads, lead, end);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (v0 + i * kThreads < vecs) {
        if constexpr (RESIDENT) kept_slice[v0 + i * kThreads] = q[i];
        float f[kN];
        Vec<T>::unpack(q[i], f);
#pragma unroll
        for (int j = 0; j < kN; ++j) m = max_nan(m, f[j]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sh.warp_sum[warp] = __float_as_uint(m);
  __syncthreads();
  if (ranks > 1) cluster_wait();
  if (tid < ranks) {
    m = __uint_as_float(static_cast<uint32_t>(sh.warp_sum[0]));
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = max_nan(m, __uint_as_float(static_cast<uint32_t>(sh.warp_sum[w])));
    *cluster.map_shared_rank(&sh.maxima[rank], tid) = m;
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
      float f[kN];
      Vec<T>::unpack(at(v), f);
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
  scale.inv_t = 1.f / temperature;
  scale.only_best = scale.best == INFINITY || scale.inv_t == INFINITY;

  float cut_logit = -INFINITY;
  uint32_t cut_index = 0xFFFFFFFFu;
  if (by_count || by_weight) {
    // The first CTA's search: first for the top-k's end, then for the top-p's.
    bool counting = by_count;  // which of the two
    uint64_t limit_count = by_count ? static_cast<uint64_t>(top_k) : 0;
    double limit_weight = 0.0;
    uint64_t cut = 0;  // rank key of the last kept token
    uint32_t base_count = 0;
    uint64_t base_weight = 0;  // before the bin or digit in question
    int bin = -1, shift = 64;
    uint64_t prefix = 0;
    bool fresh = true;  // histogram over all bins
    for (;;) {
      // A histogram: of all tokens by z, or of one bin's by the next bits of their keys.
      for (int i = tid; i < kBins; i += kThreads) hist.count[i] = hist.low[i] = hist.high[i] = 0;
      __syncthreads();
      const int next_shift = shift == 64 ? 64 - kDigitBits : max(shift - kDigitBits, 0);
      for (int v = tid; v < vecs; v += kThreads) {
        float f[kN];
        Vec<T>::unpack(at(v), f);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const uint32_t w = Scale::weight(scale.e(f[j]));
          if (w == 0) continue;
          int b = scale.bin(f[j]);
          if (!fresh) {
            if (b != bin) continue;
            const uint64_t key = rank_key(f[j], index0(v) + j);
            if (shift < 64 && (key >> shift) != prefix) continue;
            // larger keys rank first: digits count down
            b = kBins - 1 - static_cast<int>((key >> next_shift) & ((1u << (shift == 64 ? kDigitBits : shift - next_shift)) - 1u));
          }
          atomicAdd(&hist.count[b], 1u);
          const uint32_t old = atomicAdd(&hist.low[b], w);
          if (old + w < old) atomicAdd(&hist.high[b], 1u);
        }
      }
      cluster_sync(ranks);
      for (int i = rank * kThreads + tid; i < kBins; i += ranks * kThreads) {
        uint32_t c = 0;
        uint64_t w = 0;
        for (int r = 0; r < ranks; ++r) {
          const Histogram *h = cluster.map_shared_rank(&hist, r);
          c += h->count[i];
          w += (uint64_t(h->high[i]) << 32) + h->low[i];
        }
        Merged *to = cluster.map_shared_rank(&merged, 0);
        to->count[i] = c;
        to->weight[i] = w;
      }
      cluster_sync(ranks);
      bool listing = false;
      do {
        if (rank == 0) {
          // The bin where the running count or weight reaches the limit.
          uint32_t c[kBinsPerThread], cs = 0;
          uint64_t w[kBinsPerThread], ws = 0;
          if (!listing) {
#pragma unroll
            for (int i = 0; i < kBinsPerThread; ++i) {
              c[i] = merged.count[tid * kBinsPerThread + i];
              w[i] = merged.weight[tid * kBinsPerThread + i];
              cs += c[i];
              ws += w[i];
            }
          } else {
            // The listed tokens, sorted: each takes the place of a bin.
            const uint32_t n = sh.listed;
            uint32_t size = 1;
            while (size < n) size <<= 1;
            for (uint32_t i = n + tid; i < size; i += kThreads) list[i] = 0;
            __syncthreads();
            for (uint32_t span = 2; span <= size; span <<= 1) {
              for (uint32_t d = span >> 1; d > 0; d >>= 1) {
                for (uint32_t i = tid; i < size / 2; i += kThreads) {
                  const uint32_t lo = 2 * d * (i / d) + i % d, hi = lo + d;
                  const uint64_t p = list[lo], q = list[hi];
                  if ((p < q) == ((lo & span) == 0)) {
                    list[lo] = q;
                    list[hi] = p;
                  }
                }
                __syncthreads();
              }
            }
#pragma unroll
            for (int i = 0; i < kBinsPerThread; ++i) {
              const uint32_t k = tid * kBinsPerThread + i;
              c[i] = k < n ? 1u : 0u;
              w[i] = k < n ? Scale::weight(scale.e(logit_of(list[k]))) : 0u;
              cs += c[i];
              ws += w[i];
            }
          }
          uint32_t ci = cs;
          uint64_t wi = ws;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t cb = __shfl_up_sync(0xffffffffu, ci, o);
            const uint64_t wb = __shfl_up_sync(0xffffffffu, wi, o);
            if (lane >= o) {
              ci += cb;
              wi += wb;
            }
          }
          __syncthreads();
          if (lane == 31) {
            sh.warp_count[warp] = ci;
            sh.warp_sum[warp] = wi;
          }
          if (tid == 0) sh.found_bin = -1;
          __syncthreads();
          uint32_t cb = ci - cs;
          uint64_t wb = wi - ws, all = 0;
          uint32_t all_count = 0;
          for (int i = 0; i < kWarps; ++i) {
            if (i < warp) {
              cb += sh.warp_count[i];
              wb += sh.warp_sum[i];
            }
            all += sh.warp_sum[i];
            all_count += sh.warp_count[i];
          }
          // A top-k past the tokens that weigh anything cuts nothing; the top-p then follows on
          // the same histogram.
          if (counting && fresh && !listing && all_count < limit_count) {
            counting = false;
            if (by_weight) limit_weight = fmax(static_cast<double>(top_p) * static_cast<double>(all), 0.5);
          } else if (!counting && fresh && !listing && limit_weight == 0.0) {
            limit_weight = fmax(static_cast<double>(top_p) * static_cast<double>(all), 0.5);  // 0.5: the first one alone
          }
          const bool searching = counting || by_weight;
          if (searching) {
#pragma unroll
            for (int i = 0; i < kBinsPerThread; ++i) {
              const uint64_t before_c = base_count + cb, before_w = base_weight + wb;
              const bool open = counting ? before_c < limit_count : static_cast<double>(before_w) < limit_weight;
              const bool shut = counting ? before_c + c[i] >= limit_count
                                         : !(static_cast<double>(before_w + w[i]) < limit_weight);
              if (open && shut) {  // one bin of all
                sh.found_bin = tid * kBinsPerThread + i;
                sh.found_count = c[i];
                sh.found_count_before = static_cast<uint32_t>(before_c);
                sh.found_before = before_w;
                sh.total = before_w + w[i];
              }
              cb += c[i];
              wb += w[i];
            }
          }
          __syncthreads();
          Order o;
          o.command = kDone;
          o.bin = bin;
          o.shift = shift;
          o.prefix = prefix;
          const int f = sh.found_bin;
          if (searching && f >= 0) {
            if (listing) {
              cut = list[f];
              if (counting && by_weight) {
                // The top-k ends here; its weight sets the top-p's limit, from the first bin again.
                counting = false;
                limit_weight = fmax(static_cast<double>(top_p) * static_cast<double>(sh.total), 0.5);
                base_count = 0;
                base_weight = 0;
                bin = -1;
                shift = 64;
                o.command = kRefine;
                o.bin = -1;
                o.shift = 64;
              }
            } else {
              base_count = sh.found_count_before;
              base_weight = sh.found_before;
              if (fresh) {
                bin = f;
              } else {
                const int bits = shift == 64 ? kDigitBits : shift - next_shift;
                prefix = (shift == 64 ? 0 : prefix << bits) | static_cast<uint64_t>(kBins - 1 - f);
                shift = next_shift;
              }
              o.command = sh.found_count <= kList ? kGather : kRefine;
              o.bin = bin;
              o.shift = shift;
              o.prefix = prefix;
            }
          }
          o.cut_logit = cut == 0 ? -INFINITY : logit_of(cut);
          o.cut_index = cut == 0 ? 0xFFFFFFFFu : index_of(cut);
          if (tid < ranks) *cluster.map_shared_rank(&sh.order, tid) = o;
          if (tid == 0) sh.listed = 0;
        }
        cluster_sync(ranks);
        const Order o = sh.order;
        bin = o.bin;
        shift = o.shift;
        prefix = o.prefix;
        cut_logit = o.cut_logit;
        cut_index = o.cut_index;
        listing = o.command == kGather;
        if (listing) {
          uint32_t *listed = cluster.map_shared_rank(&sh.listed, 0);
          uint64_t *to = cluster.map_shared_rank(list, 0);
          for (int v = tid; v < vecs; v += kThreads) {
            float f[kN];
            Vec<T>::unpack(at(v), f);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
              if (f[j] == -INFINITY || scale.bin(f[j]) != bin || Scale::weight(scale.e(f[j])) == 0) continue;
              const uint64_t key = rank_key(f[j], index0(v) + j);
              if (shift < 64 && (key >> shift) != prefix) continue;
              const uint32_t place = atomicAdd(listed, 1u);
              if (place < kList) to[place] = key;
            }
          }
          cluster_sync(ranks);
        }
      } while (listing);
      if (sh.order.command == kDone) break;
      fresh = bin < 0;
      __syncthreads();
    }
  }

  // The kept weights of each warp's stretch of the slice, of each CTA, of the row.
  auto kept = [&](float f, uint32_t i) -> uint32_t {
    const float e = scale.e(f);
    const bool in = (f > cut_logit || (f == cut_logit && i <= cut_index)) && (e >= min_p || f == scale.best);
    return in ? Scale::weight(e) : 0u;
  };
  const int per_warp = (vecs + kThreads - 1) / kThreads * 32;
  const int begin = min(warp * per_warp, vecs), stop = min(begin + per_warp, vecs);
  uint64_t sum = 0;
  for (int v = begin + lane; v < stop; v += 32) {
    float f[kN];
    Vec<T>::unpack(at(v), f);
#pragma unroll
    for (int j = 0; j < kN; ++j) sum += kept(f[j], index0(v) + j);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) sh.warp_sum[warp] = sum;
  __syncthreads();
  if (tid < ranks) {
    uint64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += sh.warp_sum[w];
    *cluster.map_shared_rank(&sh.sums[rank], tid) = all;
  }
  cluster_sync(ranks);
  uint64_t total = 0, before = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) before = total;
    total += sh.sums[r];
  }
  for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
  const double place = floor(static_cast<double>(g.uniforms[row]) * static_cast<double>(total));
  uint64_t target = place >= 1.0 ? static_cast<uint64_t>(place) : 0;
  target = target > total - 1 ? total - 1 : target;
  if (target < before || target >= before + sum) return;  // one warp of the cluster goes on
  for (int v0 = begin; v0 < stop; v0 += 32) {
    const int v = v0 + lane;
    uint32_t w[kN];
    uint64_t mine = 0;
    if (v < stop) {
      float f[kN];
      Vec<T>::unpack(at(v), f);
#pragma unroll
      for (int j = 0; j < kN; ++j) mine += w[j] = kept(f[j], index0(v) + j);
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
  while (ranks < kMaxCluster && (row_bytes > ranks * kSliceTwoPerSm || (rows * ranks * 2 <= sms && row_bytes > ranks * 4096)))
    ranks *= 2;
  const int64_t vecs = row_bytes / 16;
  const int64_t slice = ceil_div(vecs, ranks);
  const bool resident = slice * 16 <= kSliceMost;
  TB_REQUIRE(rows * ranks <= 0x7fffffffLL && slice <= 0x7fffffffLL, TROPNN_B200_ERR_INVALID, "%s: too many rows", what);
  g.slice_vecs = static_cast<int>(slice);
  const size_t smem = kSearchBytes + 16 + (resident ? static_cast<size_t>(slice) * 16 : 0);
  const void *kernel = resident ? reinterpret_cast<const void *>(sample_kernel<T, true>)
                                : reinterpret_cast<const void *>(sample_kernel<T, false>);
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
