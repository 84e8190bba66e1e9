// Distillation of a student's logits from a teacher's top logits, mixed with the label
// cross-entropy, and its gradient.
//
// For a row s (V logits), a teacher's entries (i_k, t_k), k < K, and a label y:
//   q   = softmax(t / T) over the row's entries with an index in [0, V)
//   p   = softmax(s / T),  p1 = softmax(s)
//   loss = (1 - w) T^2 sum_k q_k (log q_k - log p_{i_k}) + w (-log p1_y)
//   dloss/ds_v = (1 - w) T (p_v - sum_{i_k = v} q_k) + w (p1_v - [v = y])
// A row without teacher entries (or without a label) drops that part; a row with neither has loss
// 0 and gradient 0 whatever its logits are.
//
// One pass over the row keeps a running maximum and the sums of exp((s - max) / T) and of
// exp(s - max); a second writes the gradient. Everything is f32, rounded once on the way out.
#include "common.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 1024;
constexpr int kPerThread = kMaxTop / kThreads;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

enum Mode { kLoss = 0, kGrad = 1, kFused = 2 };

struct DistillArgs {
  const void *logits;
  int64_t inner, outer_stride, inner_stride;  // row n at (n / inner) * outer_stride + (n % inner) * inner_stride
  int64_t vocab;
  const void *teacher;
  int teacher_dtype;
  const void *indices;
  int index_dtype;
  const int64_t *labels;
  int64_t ignore_index;
  int top;
  float inv_temperature, kl_weight, kl_grad_weight, ce_weight;  // (1-w) T^2, (1-w) T, w
  float k_t;                                                    // log2(e) / T
  // kLoss, kFused
  float *losses;
  float4 *stats;  // max, 1 / sum at T, 1 / sum at 1, 1 where the row has a target
  // kGrad, kFused: scale of row n's gradient = row_scale[n or 0] / max(count, 1)
  const float *row_scale;
  int scale_per_row;
  const float *count;
  void *grad;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float load_float(const void *p, int dtype, int64_t i) {
  if (dtype == TROPNN_B200_F32) return static_cast<const float *>(p)[i];
  if (dtype == TROPNN_B200_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ int64_t load_index(const void *p, int dtype, int64_t i) {
  return dtype == TROPNN_B200_I64 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

__device__ __forceinline__ float block_max(float v, float *shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = fmaxf(v, shared[i]);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float *shared) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v += shared[i];
  return v;
}

// Running maximum and sums of one thread.
struct Online {
  float m = kLowest, s_t = 0.f, s_1 = 0.f;
};
template <bool BOTH>
__device__ __forceinline__ void raise_max(Online &o, float m, float k_t) {
  o.s_t *= exp2_approx((o.m - m) * k_t);
  if (BOTH) o.s_1 *= exp2_approx((o.m - m) * kLog2e);
  o.m = m;
}
template <bool BOTH, int N>
__device__ __forceinline__ void take(Online &o, const float (&v)[N], float k_t) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  if (m > o.m) raise_max<BOTH>(o, m, k_t);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = v[i] - o.m;
    o.s_t += exp2_approx(d * k_t);
    if (BOTH) o.s_1 += exp2_approx(d * kLog2e);
  }
}

// Elements before the first 16-byte boundary of a row of `n`.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T *row, int64_t n) {
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(row) & 15u);
  return min64(n, off == 0 ? 0 : (16 - off) / int64_t(sizeof(T)));
}

template <typename T, int MODE, bool BOTH>
__global__ void __launch_bounds__(kThreads, 2) distill_rows_kernel(const DistillArgs g) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ float red[kThreads / 32];
  __shared__ float q_of[kMaxTop];
  __shared__ int at_of[kMaxTop];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T *x = static_cast<const T *>(g.logits) + (row / g.inner) * g.outer_stride + (row % g.inner) * g.inner_stride;

  // The row's targets; their logits come in while the row is read.
  int at[kPerThread];
  float t[kPerThread], s[kPerThread];
  float t_max = kLowest;
  bool found = false;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = tid + i * kThreads;
    at[i] = -1;
    t[i] = s[i] = 0.f;
    if (k < g.top && g.kl_weight != 0.f) {
      const int64_t v = load_index(g.indices, g.index_dtype, row * g.top + k);
      const float tv = load_float(g.teacher, g.teacher_dtype, row * g.top + k);
      if (v >= 0 && v < g.vocab && tv != -INFINITY) {
        at[i] = static_cast<int>(v);
        t[i] = tv * g.inv_temperature;
        s[i] = to_f32<T>(x[v]);
        t_max = fmaxf(t_max, t[i]);
        found = true;
      }
    }
  }
  int64_t label = -1;
  float s_label = 0.f;
  if (g.labels != nullptr && g.ce_weight != 0.f) {
    label = g.labels[row];
    if (label == g.ignore_index || label < 0 || label >= g.vocab) label = -1;
    if (label >= 0) s_label = to_f32<T>(x[label]);
  }
  const bool has_teacher = __syncthreads_or(found);
  const bool has_label = label >= 0;

  float m = 0.f, inv_t = 0.f, inv_1 = 0.f;
  if (MODE != kGrad) {
    if (has_teacher || has_label) {
      Online o;
      const int64_t head = head_of(x, g.vocab), body = (g.vocab - head) / kVec;
      if (tid < head) {
        const float v[1] = {to_f32<T>(x[tid])};
        take<BOTH>(o, v, g.k_t);
      }
      for (int64_t i = tid; i < body; i += kThreads) {
        float v[kVec];
        VecLoad<T, kVec>::load(x + head + i * kVec, v);
        take<BOTH>(o, v, g.k_t);
      }
      const int64_t tail = head + body * kVec;
      if (tail + tid < g.vocab) {
        const float v[1] = {to_f32<T>(x[tail + tid])};
        take<BOTH>(o, v, g.k_t);
      }
      m = block_max(o.m, red);
      const float s_t = block_sum(o.s_t * exp2_approx((o.m - m) * g.k_t), red);
      const float s_1 = BOTH ? block_sum(o.s_1 * exp2_approx((o.m - m) * kLog2e), red) : s_t;
      inv_t = 1.f / s_t;
      inv_1 = 1.f / s_1;
      // The losses, each difference formed from the row's maximum.
      float q_max = block_max(t_max, red), part = 0.f;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) part += at[i] >= 0 ? expf(t[i] - q_max) : 0.f;
      const float log_total = logf(block_sum(part, red)), log_s = logf(s_t);
      part = 0.f;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        if (at[i] >= 0) {
          const float log_q = t[i] - q_max - log_total, q = expf(log_q);
          if (q != 0.f) part += q * (log_q - ((s[i] - m) * g.inv_temperature - log_s));
        }
      }
      const float kl = block_sum(part, red);
      if (tid == 0) {
        float loss = has_teacher ? g.kl_weight * kl : 0.f;
        if (has_label) loss += g.ce_weight * (logf(s_1) - (s_label - m));
        g.losses[row] = loss;
        if (g.stats != nullptr) g.stats[row] = make_float4(m, inv_t, inv_1, 1.f);
      }
    } else if (tid == 0) {
      g.losses[row] = 0.f;
      if (g.stats != nullptr) g.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    const float4 st = g.stats[row];
    m = st.x;
    inv_t = st.y;
    inv_1 = st.z;
  }

  if (MODE != kLoss) {
    T *out = static_cast<T *>(g.grad) + row * g.vocab;
    float scale = g.row_scale != nullptr ? g.row_scale[g.scale_per_row ? row : 0] : 1.f;
    if (g.count != nullptr) scale /= fmaxf(*g.count, 1.f);
    const float base_t = has_teacher ? scale * g.kl_grad_weight : 0.f, base_1 = has_label ? scale * g.ce_weight : 0.f;
    const float c_t = base_t * inv_t, c_1 = base_1 * inv_1;
    auto dense = [&](float v) -> float {
      const float d = v - m;
      float r = 0.f;
      if (has_teacher) r = c_t * exp2_approx(d * g.k_t);
      if (has_label) r = fmaf(c_1, exp2_approx(d * kLog2e), r);
      return r;
    };
    const int64_t head = head_of(out, g.vocab), body = (g.vocab - head) / kVec;
    const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
    if (tid < head) out[tid] = from_f32<T>(dense(to_f32<T>(x[tid])));
    for (int64_t i = tid; i < body; i += kThreads) {
      float v[kVec];
      if (same) {
        VecLoad<T, kVec>::load(x + head + i * kVec, v);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = to_f32<T>(x[head + i * kVec + j]);
      }
      alignas(16) T w[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) w[j] = from_f32<T>(dense(v[j]));
      *reinterpret_cast<uint4 *>(out + head + i * kVec) = *reinterpret_cast<const uint4 *>(w);
    }
    const int64_t tail = head + body * kVec;
    if (tail + tid < g.vocab) out[tail + tid] = from_f32<T>(dense(to_f32<T>(x[tail + tid])));

    // The targets' own entries over it: p minus all that the teacher's entries of that index and
    // the label put there, rounded once.
    const float q_max = block_max(t_max, red);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) part += at[i] >= 0 ? expf(t[i] - q_max) : 0.f;
    const float inv_total = 1.f / block_sum(part, red);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int k = tid + i * kThreads;
      if (k < g.top) {
        at_of[k] = at[i];
        q_of[k] = at[i] >= 0 ? expf(t[i] - q_max) * inv_total : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (at[i] >= 0) {
        float q = 0.f;
        for (int k = 0; k < g.top; ++k) q += at_of[k] == at[i] ? q_of[k] : 0.f;
        const float d = s[i] - m;
        float r = base_t * (exp2_approx(d * g.k_t) * inv_t - q);
        if (has_label) r += base_1 * (exp2_approx(d * kLog2e) * inv_1 - (at[i] == label ? 1.f : 0.f));
        out[at[i]] = from_f32<T>(r);  // entries of one index write the same value
      }
    }
    if (tid == 0 && has_label) {
      bool taught = false;
      if (has_teacher)
        for (int k = 0; k < g.top; ++k) taught |= at_of[k] == label;
      if (!taught) {
        const float d = s_label - m;
        float r = base_1 * (exp2_approx(d * kLog2e) * inv_1 - 1.f);
        if (has_teacher) r += c_t * exp2_approx(d * g.k_t);
        out[label] = from_f32<T>(r);
      }
    }
  }
}

// losses summed in a fixed order; *count = rows with a target; *loss = sum, or sum / max(count, 1).
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float *losses, const float4 *stats, int64_t rows,
                                                              int mean, float *loss, float *count) {
  __shared__ float sums[32], counts[32];
  float s = 0.f, c = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    s += losses[i];
    c += stats[i].w;  // whole numbers: exact below 2^24 rows a thread
  }
  s = warp_sum(s);
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x >> 5] = s;
    counts[threadIdx.x >> 5] = c;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(sums[threadIdx.x]);
    c = warp_sum(counts[threadIdx.x]);
    if (threadIdx.x == 0) {
      *loss = mean ? s / fmaxf(c, 1.f) : s;
      *count = mean ? c : 1.f;
    }
  }
}

template <typename T, int MODE>
void launch_rows(const DistillArgs &g, int64_t rows, bool both, cudaStream_t stream) {
  if (both)
    distill_rows_kernel<T, MODE, true><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(g);
  else
    distill_rows_kernel<T, MODE, false><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(g);
}

template <int MODE>
int run_rows(const char *what, DistillArgs g, int dtype, int64_t rows, int64_t vocab, float temperature,
             float label_weight, cudaStream_t stream) {
  TB_REQUIRE(is_float_dtype(dtype), TROPNN_B200_ERR_DTYPE, "%s: logits dtype %d is not f32/f16/bf16", what, dtype);
  TB_REQUIRE(is_float_dtype(g.teacher_dtype), TROPNN_B200_ERR_DTYPE, "%s: teacher dtype %d is not f32/f16/bf16", what,
             g.teacher_dtype);
  TB_REQUIRE(g.index_dtype == TROPNN_B200_I64 || g.index_dtype == TROPNN_B200_I32, TROPNN_B200_ERR_DTYPE,
             "%s: index dtype %d is not i32/i64", what, g.index_dtype);
  TB_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && vocab >= 1 && vocab <= 0x7fffffffLL && g.inner >= 1,
             TROPNN_B200_ERR_INVALID, "%s: bad sizes (rows %lld, vocab %lld)", what, (long long)rows, (long long)vocab);
  TB_REQUIRE(g.top >= 0 && g.top <= kMaxTop, TROPNN_B200_ERR_INVALID, "%s: 0 to %d teacher entries a row, got %d", what,
             kMaxTop, g.top);
  TB_REQUIRE(temperature > 0.f && temperature < INFINITY, TROPNN_B200_ERR_INVALID,
             "%s: temperature must be positive and finite", what);
  TB_REQUIRE(label_weight >= 0.f && label_weight <= 1.f, TROPNN_B200_ERR_INVALID, "%s: label_weight must be in [0, 1]", what);
  TB_REQUIRE(label_weight == 0.f || g.labels != nullptr, TROPNN_B200_ERR_INVALID, "%s: label_weight without labels", what);
  if (rows == 0) return clear_error();
  TB_REQUIRE(g.logits != nullptr && (g.top == 0 || (g.teacher != nullptr && g.indices != nullptr)) &&
                 (MODE == kGrad || g.losses != nullptr) && (MODE == kLoss || g.grad != nullptr) &&
                 (MODE != kGrad || g.stats != nullptr),
             TROPNN_B200_ERR_INVALID, "%s: null pointer", what);
  TB_CHECK(check_current_device());
  g.vocab = vocab;
  // With the labels alone the one sum needed is the one at temperature 1.
  const float t = label_weight == 1.f ? 1.f : temperature;
  g.inv_temperature = 1.f / t;
  g.k_t = kLog2e / t;
  g.kl_weight = (1.f - label_weight) * t * t;
  g.kl_grad_weight = (1.f - label_weight) * t;
  g.ce_weight = label_weight;
  const bool both = t != 1.f && label_weight != 0.f;
  if (dtype == TROPNN_B200_F32) launch_rows<float, MODE>(g, rows, both, stream);
  else if (dtype == TROPNN_B200_F16) launch_rows<__half, MODE>(g, rows, both, stream);
  else launch_rows<__nv_bfloat16, MODE>(g, rows, both, stream);
  return check_launch(what);
}

DistillArgs make_args(const void *logits, int64_t inner, int64_t outer_stride, int64_t inner_stride, const void *teacher,
                      int teacher_dtype, const void *indices, int index_dtype, int64_t top, const int64_t *labels,
                      int64_t ignore_index) {
  DistillArgs g{};
  g.logits = logits;
  g.inner = inner;
  g.outer_stride = outer_stride;
  g.inner_stride = inner_stride;
  g.teacher = teacher;
  g.teacher_dtype = teacher_dtype;
  g.indices = indices;
  g.index_dtype = index_dtype;
  g.top = static_cast<int>(top < 0 || top > kMaxTop ? kMaxTop + 1 : top);
  g.labels = labels;
  g.ignore_index = ignore_index;
  return g;
}

}  // namespace
}  // namespace tropnn_b200

using namespace tropnn_b200;

extern "C" {

int tropnn_b200_distill_loss(const void *logits, int dtype, int64_t rows, int64_t inner, int64_t outer_stride,
                             int64_t inner_stride, int64_t vocab, const void *teacher, int teacher_dtype,
                             const void *indices, int index_dtype, int64_t top, const int64_t *labels,
                             int64_t ignore_index, float temperature, float label_weight, float *losses, float *stats,
                             void *stream) {
  DistillArgs g = make_args(logits, inner, outer_stride, inner_stride, teacher, teacher_dtype, indices, index_dtype, top,
                            labels, ignore_index);
  g.losses = losses;
  g.stats = reinterpret_cast<float4 *>(stats);
  TB_CHECK((run_rows<kLoss>("distill_loss", g, dtype, rows, vocab, temperature, label_weight, as_stream(stream))));
  return clear_error();
}

int tropnn_b200_distill_reduce(const float *losses, const float *stats, int64_t rows, int mean, float *loss, float *count,
                               void *stream) {
  TB_REQUIRE(rows >= 0, TROPNN_B200_ERR_INVALID, "distill_reduce: bad rows %lld", (long long)rows);
  TB_REQUIRE(loss != nullptr && count != nullptr && (rows == 0 || (losses != nullptr && stats != nullptr)),
             TROPNN_B200_ERR_INVALID, "distill_reduce: null pointer");
  TB_CHECK(check_current_device());
  distill_reduce_kernel<<<1, 1024, 0, as_stream(stream)>>>(losses, reinterpret_cast<const float4 *>(stats), rows, mean,
                                                           loss, count);
  TB_CHECK(check_launch("distill_reduce"));
  return clear_error();
}

int tropnn_b200_distill_grad(const void *logits, int dtype, int64_t rows, int64_t inner, int64_t outer_stride,
                             int64_t inner_stride, int64_t vocab, const void *teacher, int teacher_dtype,
                             const void *indices, int index_dtype, int64_t top, const int64_t *labels,
                             int64_t ignore_index, float temperature, float label_weight, const float *stats,
                             const float *row_scale, int scale_per_row, const float *count, void *grad, void *stream) {
  DistillArgs g = make_args(logits, inner, outer_stride, inner_stride, teacher, teacher_dtype, indices, index_dtype, top,
                            labels, ignore_index);
  g.stats = reinterpret_cast<float4 *>(const_cast<float *>(stats));
  g.row_scale = row_scale;
  g.scale_per_row = scale_per_row;
  g.count = count;
  g.grad = grad;
  TB_CHECK((run_rows<kGrad>("distill_grad", g, dtype, rows, vocab, temperature, label_weight, as_stream(stream))));
  return clear_error();
}

int tropnn_b200_distill_loss_grad(const void *logits, int dtype, int64_t rows, int64_t inner, int64_t outer_stride,
                                  int64_t inner_stride, int64_t vocab, const void *teacher, int teacher_dtype,
                                  const void *indices, int index_dtype, int64_t top, const int64_t *labels,
                                  int64_t ignore_index, float temperature, float label_weight, const float *row_scale,
                                  int scale_per_row, float *losses, void *grad, void *stream) {
  DistillArgs g = make_args(logits, inner, outer_stride, inner_stride, teacher, teacher_dtype, indices, index_dtype, top,
                            labels, ignore_index);
  g.losses = losses;
  g.row_scale = row_scale;
  g.scale_per_row = scale_per_row;
  g.grad = grad;
  TB_CHECK((run_rows<kFused>("distill_loss_grad", g, dtype, rows, vocab, temperature, label_weight, as_stream(stream))));
  return clear_error();
}

}  // extern "C"
