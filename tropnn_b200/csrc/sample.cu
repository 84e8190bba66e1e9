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
#include "common.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

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
};

__device__ __forceinline__ uint64_t rank_key(float x, int64_t i) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 ranks as +0
  const uint32_t key = b ^ ((b >> 31) != 0u ? 0xFFFFFFFFu : 0x80000000u);
  return (uint64_t(key) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float exp_of(float x, float best, float inv_t) {
  return x == best ? 1.f : expf((x - best) * inv_t);
}
__device__ __forceinline__ uint64_t weight_of(float e) { return __float2uint_rn(e * 2147483648.f); }

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t *shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWarps; ++i) v += shared[i];
  return v;
}
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t *shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWarps; ++i) v = shared[i] > v ? shared[i] : v;
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs g) {
  __shared__ uint64_t red[kWarps];
  const int64_t row = blockIdx.x, vocab = g.vocab;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T *x = static_cast<const T *>(g.logits) + (row / g.inner) * g.outer_stride + (row % g.inner) * g.inner_stride;
  const float temperature = g.temperature != nullptr ? g.temperature[row] : g.temperature_value;
  const float top_p = g.top_p != nullptr ? g.top_p[row] : g.top_p_value;
  const float min_p = g.min_p != nullptr ? g.min_p[row] : g.min_p_value;
  int64_t top_k = g.top_k_value;
  if (g.top_k != nullptr)
    top_k = g.top_k_dtype == TROPNN_B200_I64 ? static_cast<const int64_t *>(g.top_k)[row] : static_cast<const int32_t *>(g.top_k)[row];
  if (top_k <= 0 || top_k > vocab) top_k = vocab;

  uint64_t first = 0;
  bool bad = false;
  for (int64_t i = tid; i < vocab; i += kThreads) {
    const float v = ldg_f32(x + i);
    bad |= v != v;
    const uint64_t key = rank_key(v, i);
    first = key > first ? key : first;
  }
  bad = __syncthreads_or(bad);
  first = block_max(first, red);
  const uint32_t first_index = 0xFFFFFFFFu - static_cast<uint32_t>(first);
  const float best = ldg_f32(x + first_index);
  if (bad || best == -INFINITY) {
    if (tid == 0) g.tokens[row] = -1;
    return;
  }
  if (!(temperature > 0.f)) {
    if (tid == 0) g.tokens[row] = first_index;
    return;
  }
  const float inv_t = 1.f / temperature;

  auto tally = [&](uint64_t from, bool weights) -> uint64_t {  // of the tokens ranked at `from` or before
    uint64_t s = 0;
    for (int64_t i = tid; i < vocab; i += kThreads) {
      const float v = ldg_f32(x + i);
      if (rank_key(v, i) >= from) s += weights ? (v == -INFINITY ? 0 : weight_of(exp_of(v, best, inv_t))) : 1;
    }
    return block_sum(s, red);
  };
  // top-k: the largest key with k tokens at or before it.
  uint64_t cut = 0;
  if (top_k < vocab) {
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t mid = cut | (uint64_t(1) << bit);
      if (tally(mid, false) >= static_cast<uint64_t>(top_k)) cut = mid;
    }
  }
  // top-p: the smallest key whose tokens before it weigh less than the threshold.
  if (top_p < 1.f || top_p != top_p) {
    const double limit = static_cast<double>(top_p) * static_cast<double>(tally(cut, true));
    if (!(limit > 0.0)) {
      cut = first;
    } else {
      // below: the largest key k0 with weight(at or before k0) >= limit; everything past it goes.
      uint64_t last = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const uint64_t mid = last | (uint64_t(1) << bit);
        if (static_cast<double>(tally(mid > cut ? mid : cut, true)) >= limit) last = mid;
      }
      cut = last > cut ? last : cut;
    }
  }
  auto kept = [&](float v, int64_t i) -> uint64_t {
    const uint64_t key = rank_key(v, i);
    if (key == first) return weight_of(1.f);
    if (v == -INFINITY || key < cut) return 0;
    const float e = exp_of(v, best, inv_t);
    return e >= min_p ? weight_of(e) : 0;
  };
  // Each warp owns a run of the vocabulary.
  const int64_t per_warp = (vocab + kThreads - 1) / kThreads * 32;
  const int64_t begin = min64(warp * per_warp, vocab), end = min64(begin + per_warp, vocab);
  uint64_t sum = 0;
  for (int64_t i = begin + lane; i < end; i += 32) sum += kept(ldg_f32(x + i), i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = total;
    total += red[w];
  }
  const double at = floor(static_cast<double>(g.uniforms[row]) * static_cast<double>(total));
  uint64_t target = at >= 1.0 ? static_cast<uint64_t>(at) : 0;
  target = target > total - 1 ? total - 1 : target;
  if (target < before || target >= before + sum) return;  // one warp goes on
  for (int64_t i0 = begin; i0 < end; i0 += 32) {
    const int64_t i = i0 + lane;
    uint64_t upto = i < end ? kept(ldg_f32(x + i), i) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > target);
    if (past != 0) {
      if (lane == __ffs(past) - 1) g.tokens[row] = i;
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
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
  const unsigned grid = static_cast<unsigned>(rows);
  if (dtype == TROPNN_B200_F32) sample_kernel<float><<<grid, kThreads, 0, as_stream(stream)>>>(g);
  else if (dtype == TROPNN_B200_F16) sample_kernel<__half><<<grid, kThreads, 0, as_stream(stream)>>>(g);
  else sample_kernel<__nv_bfloat16><<<grid, kThreads, 0, as_stream(stream)>>>(g);
  TB_CHECK(check_launch(what));
  return clear_error();
}
