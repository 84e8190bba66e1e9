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
// The sums need the row's maximum and the gradient needs the sums, so a row is passed over twice, in
// f32 throughout and rounded once on the way out. In one call (distill_loss_grad) a cluster of up to
// 8 CTAs keeps the row in shared memory between the passes: bulk copies bring each CTA's slice, whose
// running maximum and sums are formed as the chunks arrive, one exchange through distributed shared
// memory joins them, and the gradient is written from shared memory: HBM sees one read and one write.
// Through autograd the loss kernel reads the row and the gradient kernel reads it again with the
// statistics known, each streaming through registers.
// exp2 runs on the special-function unit (16 a clock and SM), two of them an element and pass where
// T and the labels need two sums: with T = 2 the second is the square of the first. It flushes: shares of
// a row's maximum below 2^-126 are 0, in the sums as in the gradient.
//
// Measured (bf16): the loss of 8192 x 131072 335 us (6.4 TB/s, 98 % of a copy's rate), the gradient 683 us
// (6.3 TB/s), both HBM-bound; in one call 905 to 950 us by the box (4.5 to 4.7 TB/s), bound by how the
// three CTAs of an SM overlap their loads, exponentials (476 us of that unit) and stores. 4096 x 32000 with
// labels at T = 2: 56 us, 84 us and 106 us. In one call, where it took 875 us, four CTAs an SM with six
// slices a row took 975 and eight slices 1141; with the row read again instead of kept 2048 x 131072 takes
// 247 us and not 227, 1 x 131072 7.4 and not 6.6.
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kThreads = 256;  // at the row; one more warp is at the targets
constexpr int kBlock = kThreads + 32;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kChunks = 4;  // bulk copies of a slice
constexpr int kBatch = 4 * kThreads;  // vectors that the block takes at once
constexpr int64_t kSliceShared = 64 * 1024 + 64;  // bytes of a row a CTA: three CTAs on an SM
constexpr int64_t kSliceMost = 200 * 1024;        // one CTA on an SM
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

enum Mode { kLoss = 0, kGrad = 1, kFused = 2 };
// Sums an element goes into: one, two with an exponential each, two with the second the first's square.
enum Exps { kOne = 0, kTwo = 1, kSquare = 2 };

__device__ int g_distill_error = 0;

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
  float4 *stats;  // max, 1 / sum at T, 1 / sum at 1, 1 for teacher entries + 2 for a label
  // kGrad, kFused: scale of row n's gradient = row_scale[n or 0] / max(count, 1)
  const float *row_scale;
  int scale_per_row;
  const float *count;
  void *grad;
  int ranks;       // CTAs of a row
  int slice_vecs;  // 16-byte vectors of a CTA's slice
  int64_t rows;
  int rows_at_once;  // that the GPU holds
};

// Rows and `inner` are below 2^31.
template <typename T>
__device__ __forceinline__ const T *row_of(const DistillArgs &g, uint32_t row) {
  if (g.inner == 1) return static_cast<const T *>(g.logits) + row * g.outer_stride;
  const uint32_t outer = row / static_cast<uint32_t>(g.inner), rest = row - outer * static_cast<uint32_t>(g.inner);
  return static_cast<const T *>(g.logits) + outer * g.outer_stride + rest * g.inner_stride;
}

__device__ __forceinline__ float load_float(const void *p, int dtype, int64_t i) {
  if (dtype == TROPNN_B200_F32) return static_cast<const float *>(p)[i];
  if (dtype == TROPNN_B200_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ int64_t load_index(const void *p, int dtype, int64_t i) {
  return dtype == TROPNN_B200_I64 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

// 16 bytes of a row as f32 pairs.
template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  __device__ __forceinline__ static void unpack(const uint4 &q, float2 (&v)[kN / 2]) {
    if constexpr (std::is_same<T, float>::value) {
      v[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
      v[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
    } else {
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) v[i] = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
      }
    }
  }
  __device__ __forceinline__ static uint4 pack(const float2 (&v)[kN / 2]) {
    if constexpr (std::is_same<T, float>::value) {
      return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __float22half2_rn(v[i]);
          w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
          const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
          w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ static float max(const uint4 &q) {
    if constexpr (std::is_same<T, float>::value) {
      return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 *h = reinterpret_cast<const __half2 *>(&q);
      const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&q);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
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

template <typename T>
__device__ __forceinline__ uint4 nothing_vec() {  // -inf throughout
  const uint32_t w = std::is_same<T, float>::value ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}

// Vector v of the row's 16-byte grid, which starts at or before the row; elements outside the row are
// -inf (which adds nothing to a sum) and never read.
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

// The whole vectors of x's elements [e0, e1), the first 64 KB of them, on their way to L2.
//  - The gradient's CTA asks for its part before it has the statistics: 4096 x 32000 bf16 104 us without,
//    98 with 32 KB, 89 with 64 KB; at 8192 x 131072 705, 705 and 702, but 737 with 128 KB, as the CTAs there
//    ask for more than L2 holds.
//  - With a row in shared memory a CTA asks, as it begins to write, for the slice of the row that follows
//    when all rows now on the GPU are done: 8192 x 131072 bf16 918 us without, 874 with it.
//  - The loss, which is at its rows at once, does without: 58 -> 55 us at 4096 x 32000, but 34 -> 35 at
//    1000 x 50001 f16, and 64 with the row that follows.
constexpr int64_t kPrefetch = 64 * 1024;
template <typename T>
__device__ __forceinline__ void prefetch(const T *x, int64_t e0, int64_t e1) {
  const uintptr_t from = (reinterpret_cast<uintptr_t>(x + e0) + 15) & ~uintptr_t(15);
  const uintptr_t to = reinterpret_cast<uintptr_t>(x + e1) & ~uintptr_t(15);
  if (to > from) sm100::bulk_prefetch(reinterpret_cast<const void *>(from), static_cast<uint32_t>(min64(to - from, kPrefetch)));
}

// Running maximum and sums.
struct Online {
  float m = kLowest;
  float2 s_t = {0.f, 0.f}, s_1 = {0.f, 0.f};
};
template <int EXPS>
__device__ __forceinline__ float second_exp(float e, float d) {
  return EXPS == kSquare ? e * e : exp2_approx(d * kLog2e);
}
// The labels' exponentials of a vector's j-th pair, where they are not a square: the special-function
// unit, which has the teacher's to do, and the FMA pipes share them (2048 x 131072 bf16 at T = 1.5, loss
// and gradient: 342 us with all on the unit, 302 with two pairs of four, 327 with three). Which of the two
// an element gets goes by its place in its 16 bytes, so a gradient's last bits go by the row's alignment.
constexpr int kPolyPairs = 2;
__device__ __forceinline__ float2 second_pair(float2 u, int j) {
  if (j < kPolyPairs) return exp2_poly2(u);
  return make_float2(exp2_approx(u.x), exp2_approx(u.y));
}
// The first `count` of the vectors; the others are -inf.
template <typename T, int EXPS, int COUNT>
__device__ __forceinline__ void take(Online &o, const uint4 (&q)[COUNT], int count, float k_t) {
  float m = Vec<T>::max(q[0]);
#pragma unroll
  for (int i = 1; i < COUNT; ++i) m = fmaxf(m, Vec<T>::max(q[i]));
  if (m > o.m) {
    const float d = o.m - m, e = exp2_approx(d * k_t);
    o.s_t = mul2(o.s_t, both(e));
    if (EXPS != kOne) o.s_1 = mul2(o.s_1, both(second_exp<EXPS>(e, d)));
    o.m = m;
  }
  const float2 minus = both(-o.m), k = both(k_t), k1 = both(kLog2e);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if (i >= count) break;
    float2 v[Vec<T>::kN / 2];
    Vec<T>::unpack(q[i], v);
#pragma unroll
    for (int j = 0; j < Vec<T>::kN / 2; ++j) {
      const float2 d = add2(v[j], minus), t = mul2(d, k);
      const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
      o.s_t = add2(o.s_t, e);
      if (EXPS == kSquare) o.s_1 = fma2(e, e, o.s_1);
      if (EXPS == kTwo) {
        const float2 u = mul2(d, k1);
        o.s_1 = add2(o.s_1, second_pair(u, j));
      }
    }
  }
}

struct RowStats {
  float m, s_t, s_1;
};
// `a`'s sums relative to a larger maximum.
template <int EXPS>
__device__ __forceinline__ RowStats raised(RowStats a, float m, float k_t) {
  const float d = a.m - m, e = exp2_approx(d * k_t);
  return {m, a.s_t * e, EXPS == kOne ? 0.f : a.s_1 * second_exp<EXPS>(e, d)};
}
// All of the lanes' (of the first WIDTH lanes', in each group of WIDTH) statistics together.
template <int EXPS, int WIDTH>
__device__ __forceinline__ RowStats joined(RowStats a, float k_t) {
  float m = a.m;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  a = raised<EXPS>(a, m, k_t);
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    a.s_t += __shfl_xor_sync(0xffffffffu, a.s_t, o);
    if (EXPS != kOne) a.s_1 += __shfl_xor_sync(0xffffffffu, a.s_1, o);
  }
  if (EXPS == kOne) a.s_1 = a.s_t;
  return a;
}

// A row's targets. Up to 128 entries of the teacher are read by a warp of its own while the others are at
// the row; of more, warp w reads [128 w, 128 w + 128) before its share of the row. After the barrier
// that the row's sums take anyway, each thread has the parts at hand.
constexpr int kEntriesPerWarp = kMaxTop / kWarps, kEntriesPerLane = kEntriesPerWarp / 32;
struct TeacherPart {
  float t_max, total;         // sum of e = exp((t - t_max) / T)
  float entropy, cross, from; // sums of e (t - t_max) / T and of e (s - from) / T
  int count;                  // of its entries in the CTA's part of the row
};
struct EntryTable {
  alignas(16) int at[kMaxTop];   // -1: none
  alignas(16) float q[kMaxTop];  // t, later its share exp((t - t_max) / T) / total
  uint16_t mine[kMaxTop];        // numbers of the entries in the CTA's part, a stretch a warp
  TeacherPart part[kWarps];
  int label;  // -1: none
  float s_label;
};

template <typename T>
__device__ __forceinline__ void load_targets(const DistillArgs &g, int64_t row, const T *x, int64_t e0, int64_t e1,
                                             bool for_loss, EntryTable &table) {
  const int lane = threadIdx.x & 31;
  const int top = g.kl_weight != 0.f ? g.top : 0;
  const int warp = static_cast<int>(threadIdx.x >> 5) - (top <= kEntriesPerWarp ? kWarps : 0);
  const int base = warp * kEntriesPerWarp;
  if (warp < 0 || base >= max(top, 1)) return;
  int64_t label = -1;
  if (warp == 0 && g.labels != nullptr && g.ce_weight != 0.f) label = g.labels[row];
  int64_t at[kEntriesPerLane];
  float t[kEntriesPerLane], s[kEntriesPerLane];
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    const int k = base + i * 32 + lane;
    at[i] = -1;
    t[i] = 0.f;
    if (k < top) {
      at[i] = load_index(g.indices, g.index_dtype, row * g.top + k);
      t[i] = load_float(g.teacher, g.teacher_dtype, row * g.top + k);
    }
  }
  if (label == g.ignore_index || label < 0 || label >= g.vocab) label = -1;
  float s_label = 0.f;
  if (for_loss && label >= 0) s_label = to_f32<T>(x[label]);
  TeacherPart p = {kLowest, 0.f, 0.f, 0.f, -INFINITY, 0};
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    s[i] = -INFINITY;
    if (at[i] < 0 || at[i] >= g.vocab || t[i] == -INFINITY) at[i] = -1;
    if (at[i] >= 0) {
      p.t_max = fmaxf(p.t_max, t[i]);
      if (for_loss) s[i] = to_f32<T>(x[at[i]]);
    }
  }
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    const int k = base + i * 32 + lane;
    if (base + i * 32 < top) {
      table.at[k] = static_cast<int>(at[i]);
      table.q[k] = t[i];
      const bool here = at[i] >= e0 && at[i] < e1;
      const uint32_t all = __ballot_sync(0xffffffffu, here);
      if (here) table.mine[base + p.count + __popc(all & ((1u << lane) - 1u))] = static_cast<uint16_t>(k);
      p.count += __popc(all);
    }
    p.from = fmaxf(p.from, s[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    p.t_max = fmaxf(p.t_max, __shfl_xor_sync(0xffffffffu, p.t_max, o));
    p.from = fmaxf(p.from, __shfl_xor_sync(0xffffffffu, p.from, o));
  }
  if (p.from == -INFINITY) p.from = 0.f;
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    if (at[i] >= 0) {
      const float d = (t[i] - p.t_max) * g.inv_temperature, e = expf(d);
      p.total += e;
      if (e != 0.f) {
        p.entropy += e * d;
        p.cross += e * ((s[i] - p.from) * g.inv_temperature);
      }
    }
  }
  p.total = warp_sum(p.total);
  p.entropy = warp_sum(p.entropy);
  p.cross = warp_sum(p.cross);
  if (lane == 0) {
    table.part[warp] = p;
    if (warp == 0) {
      table.label = static_cast<int>(label);
      table.s_label = s_label;
    }
  }
}
// The parts together, after a barrier.
struct Teacher {
  int parts;  // 0: no entries
  float t_max, total;
  __device__ __forceinline__ Teacher(const DistillArgs &g, const EntryTable &table) {
    parts = g.kl_weight != 0.f ? (g.top + kEntriesPerWarp - 1) / kEntriesPerWarp : 0;
    t_max = kLowest;
    total = 0.f;
    for (int w = 0; w < parts; ++w) t_max = fmaxf(t_max, table.part[w].t_max);
    for (int w = 0; w < parts; ++w) total += table.part[w].total * expf((table.part[w].t_max - t_max) * g.inv_temperature);
    if (total == 0.f) parts = 0;  // NaN stays
  }
};
__device__ __forceinline__ float teacher_loss(const DistillArgs &g, const EntryTable &table, const Teacher &teacher, float m,
                                              float s_t) {
  float entropy = 0.f, cross = 0.f;
  for (int w = 0; w < teacher.parts; ++w) {
    const TeacherPart &p = table.part[w];
    const float d = (p.t_max - teacher.t_max) * g.inv_temperature, f = expf(d);
    if (p.total == 0.f || f == 0.f) continue;  // no part of the sum, however far off d or the logits are
    entropy += f * (p.entropy + p.total * d);
    cross += f * (p.cross + p.total * ((p.from - m) * g.inv_temperature));
  }
  return (entropy - cross) / teacher.total - logf(teacher.total) + logf(s_t);
}
// Entries become shares, all threads; a barrier has to follow.
__device__ __forceinline__ void form_shares(const DistillArgs &g, const Teacher &teacher, EntryTable &table) {
  if (teacher.parts == 0) return;
  const float inv_total = 1.f / teacher.total;
  for (int k = threadIdx.x; k < (g.top + 31 & ~31); k += kBlock)
    table.q[k] = table.at[k] >= 0 ? expf((table.q[k] - teacher.t_max) * g.inv_temperature) * inv_total : 0.f;
}

struct GradScale {
  float base_t, base_1;  // scale (1 - w) T and scale w, 0 without such a target
  float c_t, c_1;        // the same over the sums
};
__device__ __forceinline__ float scale_of(const DistillArgs &g, int64_t row) {
  float scale = g.row_scale != nullptr ? g.row_scale[g.scale_per_row ? row : 0] : 1.f;
  if (g.count != nullptr) scale /= fmaxf(*g.count, 1.f);
  return scale;
}
__device__ __forceinline__ GradScale grad_scale(const DistillArgs &g, bool has_teacher, bool has_label, float scale,
                                                float inv_t, float inv_1) {
  GradScale c;
  c.base_t = has_teacher ? scale * g.kl_grad_weight : 0.f;
  c.base_1 = has_label ? scale * g.ce_weight : 0.f;
  c.c_t = has_teacher ? c.base_t * inv_t : 0.f;
  c.c_1 = has_label ? c.base_1 * inv_1 : 0.f;
  return c;
}
template <int EXPS>
__device__ __forceinline__ float2 dense2(float2 v, float m, float k_t, const GradScale &c, int j) {
  const float2 d = add2(v, both(-m)), t = mul2(d, both(k_t));
  const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
  if (EXPS == kOne) return mul2(e, both(c.c_t + c.c_1));
  if (EXPS == kSquare) return mul2(e, fma2(e, both(c.c_1), both(c.c_t)));
  const float2 u = mul2(d, both(kLog2e));
  return fma2(second_pair(u, j), both(c.c_1), mul2(e, both(c.c_t)));
}
// The dense part of the gradient of a row's elements [e0, e1). vec_at gives vectors of the input where
// it is aligned as the output, element_at any element.
template <typename T, int EXPS, typename VecAt, typename ElementAt>
__device__ __forceinline__ void write_dense(T *out, int64_t e0, int64_t e1, bool alike, float m, float k_t,
                                            const GradScale &c, VecAt vec_at, ElementAt element_at) {
  constexpr int kN = Vec<T>::kN, kAhead = 4;
  const int tid = threadIdx.x;
  if (tid >= kThreads) return;
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out + e0) & 15u);
  const int64_t head = min64(e1 - e0, off == 0 ? 0 : (16 - off) / int64_t(sizeof(T)));
  const int64_t start = e0 + head, tail = start + (e1 - start) / kN * kN;
  const int body = static_cast<int>((tail - start) / kN);
  auto one = [&](int64_t e) { out[e] = from_f32<T>(dense2<EXPS>(both(element_at(e)), m, k_t, c, kN).x); };
  auto put = [&](int i, float2 (&v)[kN / 2]) {
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) v[j] = dense2<EXPS>(v[j], m, k_t, c, j);
    __stcs(reinterpret_cast<uint4 *>(out + start) + i, Vec<T>::pack(v));
  };
  if (tid < head) one(e0 + tid);
  if (alike) {
    for (int i = tid; i < body; i += kAhead * kThreads) {
      uint4 q[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        if (i + n * kThreads < body) q[n] = vec_at(start, i + n * kThreads);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        if (i + n * kThreads >= body) break;
        float2 v[kN / 2];
        Vec<T>::unpack(q[n], v);
        put(i + n * kThreads, v);
      }
    }
  } else {
    for (int i = tid; i < body; i += kThreads) {
      float2 v[kN / 2];
#pragma unroll
      for (int j = 0; j < kN / 2; ++j) {
        const int64_t e = start + int64_t(i) * kN + 2 * j;
        v[j] = make_float2(element_at(e), element_at(e + 1));
      }
      put(i, v);
    }
  }
  if (tail + tid < e1) one(tail + tid);
}
template <typename T>
__device__ __forceinline__ void write_zeros(T *out, int64_t e0, int64_t e1) {
  constexpr int kN = Vec<T>::kN;
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out + e0) & 15u);
  const int64_t head = min64(e1 - e0, off == 0 ? 0 : (16 - off) / int64_t(sizeof(T)));
  const int64_t start = e0 + head, tail = start + (e1 - start) / kN * kN;
  if (int64_t(threadIdx.x) < head) out[e0 + threadIdx.x] = from_f32<T>(0.f);
  for (int64_t e = start + threadIdx.x * kN; e < tail; e += kBlock * kN) __stcs(reinterpret_cast<uint4 *>(out + e), make_uint4(0, 0, 0, 0));
  if (tail + threadIdx.x < e1) out[tail + threadIdx.x] = from_f32<T>(0.f);
}
// The targets of the part over it: p minus all that the teacher's entries of that index and the label
// put there, rounded once. After a barrier that follows write_dense and form_shares; every thread takes
// part.
template <typename T, int EXPS, typename ElementAt>
__device__ __forceinline__ void write_targets(const DistillArgs &g, T *out, int64_t e0, int64_t e1, float m, const GradScale &c,
                                              const EntryTable &table, int parts, ElementAt element_at) {
  const int tid = threadIdx.x, padded = parts > 0 ? g.top + 3 & ~3 : 0, label = table.label;
  auto sum_at = [&](int e, bool &found) -> float {  // in the entries' order
    float q = 0.f;
    for (int k = 0; k < padded; k += 4) {
      const int4 a = *reinterpret_cast<const int4 *>(&table.at[k]);
      const float4 v = *reinterpret_cast<const float4 *>(&table.q[k]);
      q += a.x == e ? v.x : 0.f;
      q += a.y == e ? v.y : 0.f;
      q += a.z == e ? v.z : 0.f;
      q += a.w == e ? v.w : 0.f;
      found |= a.x == e || a.y == e || a.z == e || a.w == e;
    }
    return q;
  };
  auto put = [&](int e, float q) {
    const float p = dense2<EXPS>(both(element_at(e)), m, g.k_t, c, kMaxTop).x;
    out[e] = from_f32<T>(p - c.base_t * q - (e == label ? c.base_1 : 0.f));
  };
  if (tid >= kThreads) return;
  bool found = false;
  // The warps' stretches of entries are spread over the block one after the other.
  int before = 0;
  for (int w = 0; w < parts; ++w) {
    const int count = table.part[w].count;
    for (int i = (tid - before) & (kThreads - 1); i < count; i += kThreads) {
      const int e = table.at[table.mine[w * kEntriesPerWarp + i]];
      put(e, sum_at(e, found));  // entries of one index write the same value
    }
    before += count;
  }
  if (tid == kThreads - 1 && label >= e0 && label < e1) {
    found = false;
    const float q = sum_at(label, found);
    if (!found) put(label, q);
  }
}

// Loss (MODE kLoss), or loss and gradient (kFused), of a row a cluster. RESIDENT: the slice stays in
// shared memory for the gradient; else it is read again.
template <typename T, int MODE, int EXPS, bool RESIDENT>
__global__ void __launch_bounds__(kBlock, RESIDENT ? 3 : 4) distill_row_kernel(const DistillArgs g) {
  constexpr int kN = Vec<T>::kN;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ RowStats of_warp[kWarps], of_rank[kMaxCluster];
  __shared__ EntryTable table;
  __shared__ uint64_t full[kChunks];
  __shared__ int abort;
  uint4 *slice = reinterpret_cast<uint4 *>(dynamic);
  const uint32_t row32 = blockIdx.x / static_cast<uint32_t>(g.ranks);
  const int rank = static_cast<int>(blockIdx.x - row32 * g.ranks);
  const int64_t row = row32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T *x = row_of<T>(g, row32);
  const int64_t lead = static_cast<int64_t>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)), end = lead + g.vocab;
  const T *grid = x - lead;
  const int64_t vec0 = int64_t(rank) * g.slice_vecs;
  const int vecs = static_cast<int>(min64(g.slice_vecs, max(int64_t(0), (end + kN - 1) / kN - vec0)));
  const int64_t e0 = max(int64_t(0), vec0 * kN - lead), e1 = max(e0, min64(g.vocab, (vec0 + vecs) * kN - lead));
  if (g.ranks > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  // Whole vectors of the slice come as bulk copies; one at either end of the row may be cut.
  const bool first_cut = vec0 == 0 && lead > 0, last_cut = vec0 + vecs == (end + kN - 1) / kN && end % kN != 0;
  const int whole0 = first_cut ? 1 : 0, whole1 = max(vecs - (last_cut ? 1 : 0), whole0);
  // Chunks are whole batches of the block, so that kernels with and without them sum up alike.
  const int per_chunk = (whole1 - whole0 + kChunks * kBatch - 1) / (kChunks * kBatch) * kBatch;
  if (RESIDENT) {
    if (tid == 0) {
      abort = 0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) sm100::mbar_init(&full[c], 1);
      sm100::mbar_init_fence();
      sm100::fence_proxy_async_smem();
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int from = min(whole0 + c * per_chunk, whole1), to = min(from + per_chunk, whole1);
        if (to > from) {
          sm100::mbar_expect_tx(&full[c], (to - from) * 16);
          sm100::bulk_load_1d(slice + from, grid + (vec0 + from) * kN, (to - from) * 16, &full[c]);
        }
      }
    }
    __syncthreads();  // the barriers are set up
  }
  const float scale = MODE == kFused ? scale_of(g, row) : 1.f;
  load_targets<T>(g, row, x, e0, e1, rank == 0, table);

  // One order of summation for the kernels that split a row alike: cut vectors first, then batch by batch
  // (how many CTAs a row has goes by the call and by the number of rows). A row without a target is summed
  // up too, and nothing made of it.
  Online o;
  if (tid == kThreads - 1) {
    if (first_cut && vecs > 0) {
      const uint4 q[1] = {load_vec<T>(grid, vec0, lead, end)};
      if (RESIDENT) slice[0] = q[0];
      take<T, EXPS>(o, q, 1, g.k_t);
    }
    if (last_cut && vecs > whole0) {
      const uint4 q[1] = {load_vec<T>(grid, vec0 + vecs - 1, lead, end)};
      if (RESIDENT) slice[vecs - 1] = q[0];
      take<T, EXPS>(o, q, 1, g.k_t);
    }
  }
  const uint4 *whole = RESIDENT ? slice : reinterpret_cast<const uint4 *>(grid) + vec0;
  const uint4 nothing = nothing_vec<T>();
  if (warp < kWarps) {
    for (int from = whole0, c = 0; from < whole1; from += per_chunk, ++c) {
      const int to = min(from + per_chunk, whole1);
      if (RESIDENT && !sm100::mbar_wait(&full[c], 0, &abort, &g_distill_error)) break;
      int v = from + tid;
      // Full batches without checks where a slice is in shared memory: 2048 x 131072 bf16 at T = 2 243 ->
      // 235 us. From global memory two loops cost registers: the loss of 4096 x 32000 56.5 -> 59 us.
      for (; RESIDENT && v + 3 * kThreads < to; v += kBatch) {
        uint4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = whole[v + i * kThreads];
        take<T, EXPS>(o, q, 4, g.k_t);
      }
      for (; v < to; v += kBatch) {
        uint4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q[i] = nothing;
          if (v + i * kThreads < to) q[i] = RESIDENT ? whole[v + i * kThreads] : __ldg(whole + v + i * kThreads);
        }
        take<T, EXPS>(o, q, (to - v + kThreads - 1) / kThreads, g.k_t);
      }
    }
    const RowStats mine = joined<EXPS, 32>({o.m, o.s_t.x + o.s_t.y, o.s_1.x + o.s_1.y}, g.k_t);
    if (lane == 0) of_warp[warp] = mine;
  }
  __syncthreads();
  RowStats st;
  st = joined<EXPS, kWarps>(of_warp[lane % kWarps], g.k_t);
  if (g.ranks > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // all have started
    if (tid < g.ranks) *cooperative_groups::this_cluster().map_shared_rank(&of_rank[rank], tid) = st;
    cooperative_groups::this_cluster().sync();
    const RowStats none = {kLowest, 0.f, 0.f};
    st = joined<EXPS, kMaxCluster>(lane % kMaxCluster < g.ranks ? of_rank[lane % kMaxCluster] : none, g.k_t);
  }
  const float inv_t = 1.f / st.s_t, inv_1 = 1.f / st.s_1;
  const Teacher teacher(g, table);
  const bool has_teacher = teacher.parts > 0, has_label = table.label >= 0;
  if constexpr (MODE == kFused) {
    T *out = static_cast<T *>(g.grad) + row * g.vocab;
    if (RESIDENT && tid == kThreads && row + g.rows_at_once < g.rows)
      prefetch<T>(row_of<T>(g, row32 + g.rows_at_once), e0, e1);
    if (has_teacher || has_label) {
      const GradScale c = grad_scale(g, has_teacher, has_label, scale, inv_t, inv_1);
      const bool alike = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
      auto vec_at = [&](int64_t start, int i) -> uint4 {
        if constexpr (RESIDENT) return slice[static_cast<int>((start + lead) / kN - vec0) + i];
        else return __ldg(reinterpret_cast<const uint4 *>(x + start) + i);
      };
      auto element_at = [&](int64_t e) -> float {
        if constexpr (RESIDENT) return to_f32<T>(reinterpret_cast<const T *>(slice)[e + lead - vec0 * kN]);
        else return ldg_f32(x + e);
      };
      form_shares(g, teacher, table);
      write_dense<T, EXPS>(out, e0, e1, alike, st.m, g.k_t, c, vec_at, element_at);
      __syncthreads();
      write_targets<T, EXPS>(g, out, e0, e1, st.m, c, table, teacher.parts, element_at);
    } else {
      write_zeros<T>(out, e0, e1);
    }
  }
  if (rank == 0 && tid == 0) {
    float loss = 0.f;
    if (has_teacher) loss = g.kl_weight * teacher_loss(g, table, teacher, st.m, st.s_t);
    if (has_label) loss += g.ce_weight * (logf(st.s_1) - (table.s_label - st.m));
    g.losses[row] = loss;
    if (MODE == kLoss && g.stats != nullptr)
      g.stats[row] = make_float4(st.m, inv_t, inv_1, static_cast<float>((has_teacher ? 1 : 0) + (has_label ? 2 : 0)));
  }
  if (RESIDENT && tid == kThreads && abort != 0) {  // a wait ran out: the copies are seen out first
    for (int from = whole0, c = 0; from < whole1; from += per_chunk, ++c) sm100::mbar_drain(&full[c], 0);
  }
}

// The gradient from the loss's statistics: each CTA a part of a row.
template <typename T, int EXPS>
__global__ void __launch_bounds__(kBlock, 4) distill_grad_kernel(const DistillArgs g) {
  constexpr int kN = Vec<T>::kN;
  __shared__ EntryTable table;
  const uint32_t row32 = blockIdx.x / static_cast<uint32_t>(g.ranks);
  const int64_t row = row32, part = blockIdx.x - row32 * g.ranks;
  const T *x = row_of<T>(g, row32);
  T *out = static_cast<T *>(g.grad) + row * g.vocab;
  // Parts end on the output's 16-byte grid.
  const int64_t lead = static_cast<int64_t>((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
  const int64_t e0 = max(int64_t(0), part * g.slice_vecs * kN - lead);
  const int64_t e1 = max(e0, min64(g.vocab, (part + 1) * g.slice_vecs * kN - lead));
  if (threadIdx.x == kThreads) prefetch<T>(x, e0, e1);
  const float4 st = g.stats[row];
  const int has = static_cast<int>(st.w);
  if (has == 0) {
    write_zeros<T>(out, e0, e1);
    return;
  }
  load_targets<T>(g, row, x, e0, e1, false, table);
  const GradScale c = grad_scale(g, (has & 1) != 0, (has & 2) != 0, scale_of(g, row), st.y, st.z);
  const bool alike = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
  auto vec_at = [&](int64_t start, int i) -> uint4 { return __ldg(reinterpret_cast<const uint4 *>(x + start) + i); };
  auto element_at = [&](int64_t e) -> float { return ldg_f32(x + e); };
  write_dense<T, EXPS>(out, e0, e1, alike, st.x, g.k_t, c, vec_at, element_at);
  __syncthreads();
  const Teacher teacher(g, table);
  form_shares(g, teacher, table);
  __syncthreads();
  write_targets<T, EXPS>(g, out, e0, e1, st.x, c, table, teacher.parts, element_at);
}

// losses summed in a fixed order; *count = rows with a target; *loss = sum, or sum / max(count, 1).
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float *losses, const float4 *stats, int64_t rows,
                                                              int mean, float *loss, float *count) {
  __shared__ float sums[32], counts[32];
  float s = 0.f, c = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    s += losses[i];
    c += stats[i].w > 0.f ? 1.f : 0.f;  // whole numbers: exact below 2^24 rows a thread
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

// CTAs an SM up to which a row is split further. 16 x 131072 bf16, split and not: loss 6.9 and 13.6 us,
// gradient 4.9 and 12.1 us (148 rows 17 and 23 us), in one call 8.0 and 9.0 us.
template <int MODE>
constexpr int kIdle = MODE == kGrad ? 4 : 1;

template <typename T, int MODE, int EXPS>
int launch_rows(const char *what, DistillArgs g, int64_t rows, cudaStream_t stream) {
  int sms = 0;
  TB_CHECK(sm100::sm_count(&sms));
  // In one call: the fewest CTAs a row that keep its slices at three CTAs an SM. Loss or gradient alone:
  // a CTA a row. More of them while SMs are idle.
  const int64_t row_bytes = g.vocab * int64_t(sizeof(T)) + 32;
  const int64_t most = MODE == kFused ? kSliceShared : int64_t(1) << 40;
  int ranks = 1;
  while (ranks < kMaxCluster && (row_bytes > ranks * most || (rows * ranks * 2 <= kIdle<MODE> * sms && row_bytes > ranks * 8192)))
    ranks *= 2;
  const int64_t slice = ceil_div(row_bytes / 16, ranks);
  TB_REQUIRE(rows * ranks <= 0x7fffffffLL && slice <= 0x7fffffffLL, TROPNN_B200_ERR_INVALID, "%s: too many rows", what);
  g.ranks = ranks;
  g.slice_vecs = static_cast<int>(slice);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  config.blockDim = dim3(kBlock);
  config.stream = stream;
  const void *kernel = nullptr;
  cudaLaunchAttribute attr{};
  if constexpr (MODE == kGrad) {
    kernel = reinterpret_cast<const void *>(distill_grad_kernel<T, EXPS>);
  } else {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(ranks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    kernel = reinterpret_cast<const void *>(distill_row_kernel<T, MODE, EXPS, false>);
    if constexpr (MODE == kFused) {
      if (slice * 16 <= kSliceMost) {
        kernel = reinterpret_cast<const void *>(distill_row_kernel<T, MODE, EXPS, true>);
        g.rows = rows;
        g.rows_at_once = std::max(1, (slice * 16 <= kSliceShared ? 3 : 1) * sms / ranks);
        config.dynamicSmemBytes = static_cast<size_t>(slice) * 16;
        // The static tables count too: above 48 KB in all the kernel has to be told.
        TB_CHECK(ensure_dynamic_smem(kernel, std::max<size_t>(config.dynamicSmemBytes, 49 * 1024), what));
      }
    }
  }
  void *args[] = {&g};
  cudaLaunchKernelExC(&config, kernel, args);
  return check_launch(what);
}
template <typename T, int MODE>
int launch_exps(const char *what, const DistillArgs &g, int64_t rows, int exps, cudaStream_t stream) {
  if (exps == kOne) return launch_rows<T, MODE, kOne>(what, g, rows, stream);
  if (exps == kTwo) return launch_rows<T, MODE, kTwo>(what, g, rows, stream);
  return launch_rows<T, MODE, kSquare>(what, g, rows, stream);
}

template <int MODE>
int run_rows(const char *what, DistillArgs g, int dtype, int64_t rows, int64_t vocab, float temperature,
             float label_weight, cudaStream_t stream) {
  TB_REQUIRE(is_float_dtype(dtype), TROPNN_B200_ERR_DTYPE, "%s: logits dtype %d is not f32/f16/bf16", what, dtype);
  TB_REQUIRE(is_float_dtype(g.teacher_dtype), TROPNN_B200_ERR_DTYPE, "%s: teacher dtype %d is not f32/f16/bf16", what,
             g.teacher_dtype);
  TB_REQUIRE(g.index_dtype == TROPNN_B200_I64 || g.index_dtype == TROPNN_B200_I32, TROPNN_B200_ERR_DTYPE,
             "%s: index dtype %d is not i32/i64", what, g.index_dtype);
  TB_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && vocab >= 1 && vocab <= 0x7fffffffLL && g.inner >= 1 && g.inner <= 0x7fffffffLL,
             TROPNN_B200_ERR_INVALID, "%s: bad sizes (rows %lld, vocab %lld)", what, (long long)rows, (long long)vocab);
  TB_REQUIRE(g.top >= 0 && g.top <= kMaxTop, TROPNN_B200_ERR_INVALID, "%s: 0 to %d teacher entries a row, got %d", what,
             kMaxTop, g.top);
  TB_REQUIRE(temperature > 0.f && temperature < INFINITY, TROPNN_B200_ERR_INVALID,
             "%s: temperature must be positive and finite", what);
  // f32 holds 1 / T and (1 - w) T^2 with room for what they multiply.
  TB_REQUIRE(label_weight == 1.f || (temperature >= 0x1p-60f && temperature <= 0x1p60f), TROPNN_B200_ERR_INVALID,
             "%s: temperature must be in [2^-60, 2^60] for a teacher", what);
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
  const int exps = t == 1.f || label_weight == 0.f ? kOne : t == 2.f ? kSquare : kTwo;
  if (dtype == TROPNN_B200_F32) return launch_exps<float, MODE>(what, g, rows, exps, stream);
  if (dtype == TROPNN_B200_F16) return launch_exps<__half, MODE>(what, g, rows, exps, stream);
  return launch_exps<__nv_bfloat16, MODE>(what, g, rows, exps, stream);
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

// Reads and clears this file's device error word (a wait for a bulk copy that ran out).
int read_distill_error(int *value) {
  int v = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&v, g_distill_error, sizeof(int));
  if (err != cudaSuccess)
    return set_error(TROPNN_B200_ERR_LAUNCH, "reading the device error word: %s", cudaGetErrorString(err));
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_distill_error, &zero, sizeof(int));
  }
  *value = v;
  return TROPNN_B200_OK;
}

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
