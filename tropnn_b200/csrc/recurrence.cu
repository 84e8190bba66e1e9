// Gated linear recurrence over token sequences: forward, backward and the single-token step.
//
//   a_t = sigmoid(f_t), c_t = 1 - a_t = sigmoid(-f_t)          (per channel)
//   h_t = keep_t a_t h_{t-1} + c_t x_t                          (keep_t = 0 at a reset, else 1)
//
// The recurrence is linear, so a run of steps maps the state before it to P h + H with P the
// product of its keep_t a_t. A warp owns kRun consecutive steps of 64 channels (two a lane): it
// scans them in registers from h = 0 for (P, H), hands those to the other warps through shared
// memory, composes the runs before its own into its incoming state and scans again from there.
// A tile is 8 warps' runs; a CTA walks the tiles of its 64 channels in order. One read of gate
// and value, one write of h: the kernels are bound by HBM traffic.
#include "common.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChan = 64;                    // channels of a CTA, two a lane
constexpr int kRunFwd = 16;                  // steps of a warp's run, forward
constexpr int kRunBwd = 8;                   // ... backward (more live values a step)
constexpr int kTileFwd = kWarps * kRunFwd;   // 128
constexpr int kTileBwd = kWarps * kRunBwd;   // 64: also the distance of the saved states
static_assert(kTileFwd % kTileBwd == 0 && kTileBwd % kRunFwd == 0, "saved states start at a run of the forward");

// Two channels of one step as they lie in memory.
template <typename T>
struct Raw {
  uint32_t v;
};
template <>
struct Raw<float> {
  float a, b;
};

// The second channel of a lane: the next one where rows allow paired accesses, else 32 on, so
// that single-element accesses of a warp stay consecutive.
template <bool PAIRED>
__device__ __forceinline__ int first_channel(int lane) { return PAIRED ? 2 * lane : lane; }
template <bool PAIRED>
constexpr int kSecond = PAIRED ? 1 : 32;

template <typename T, bool PAIRED>
__device__ __forceinline__ Raw<T> load_raw(const T *p, bool on0, bool on1) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = r.b = 0.f;
    if constexpr (PAIRED) {
      if (on0) {
        const float2 q = __ldg(reinterpret_cast<const float2 *>(p));
        r.a = q.x;
        r.b = q.y;
      }
    } else {
      if (on0) r.a = __ldg(p);
      if (on1) r.b = __ldg(p + 32);
    }
  } else {
    r.v = 0u;
    if constexpr (PAIRED) {
      if (on0) r.v = __ldg(reinterpret_cast<const unsigned int *>(p));
    } else {
      const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
      uint32_t lo = 0, hi = 0;
      if (on0) lo = __ldg(u);
      if (on1) hi = __ldg(u + 32);
      r.v = lo | (hi << 16);
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ float2 unpack(Raw<T> r) {
  if constexpr (std::is_same<T, float>::value) {
    return make_float2(r.a, r.b);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&r.v));
  } else {
    return make_float2(__uint_as_float(r.v << 16), __uint_as_float(r.v & 0xFFFF0000u));
  }
}

template <typename T, bool PAIRED>
__device__ __forceinline__ void store_pair(T *p, float2 v, bool on0, bool on1) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (PAIRED) {
      if (on0) *reinterpret_cast<float2 *>(p) = v;
    } else {
      if (on0) p[0] = v.x;
      if (on1) p[32] = v.y;
    }
  } else {
    const T a = from_f32<T>(v.x), b = from_f32<T>(v.y);
    if constexpr (PAIRED) {
      const uint32_t w = uint32_t(*reinterpret_cast<const unsigned short *>(&a)) |
                         (uint32_t(*reinterpret_cast<const unsigned short *>(&b)) << 16);
      if (on0) *reinterpret_cast<uint32_t *>(p) = w;
    } else {
      if (on0) p[0] = a;
      if (on1) p[32] = b;
    }
  }
}

// a and c = 1 - a. The smaller one, m = e / (1 + e) with e = exp(-|f|), has its full relative
// accuracy; the larger is 1 - m, the f32 next to it.
__device__ __forceinline__ void gates(float f, float &a, float &c) {
  const float e = __expf(-fabsf(f));
  const float m = __fdividef(e, 1.f + e), o = 1.f - m;
  a = f < 0.f ? m : o;
  c = f < 0.f ? o : m;
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) { return make_float2(x.x * y.x, x.y * y.y); }
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  return make_float2(fmaf(x.x, y.x, z.x), fmaf(x.y, y.y, z.y));
}

// P h + H; a run that a reset cut (P = 0) takes nothing of h, not even an infinity's NaN.
__device__ __forceinline__ float2 apply_run(float2 p, float2 h, float2 add) {
  return make_float2(p.x == 0.f ? add.x : fmaf(p.x, h.x, add.x), p.y == 0.f ? add.y : fmaf(p.y, h.y, add.y));
}

struct RecurrenceArgs {
  const void *gate, *value;
  int64_t gate_batch, gate_step, value_batch, value_step;
  const float *h0;
  const uint8_t *reset;
  int64_t steps, dim;
  int channel_blocks;
  void *h;
  float *h_last;
  float *saved;  // [batch, saved_tiles, dim]: the state before each 64-step tile; NULL: not kept
  int64_t saved_tiles;
  // backward
  const void *grad;
  const float *grad_last;
  void *grad_gate, *grad_value;
  float *grad_h0;
};

// The reset flags of `n` consecutive steps as bits.
__device__ __forceinline__ uint32_t reset_bits(const uint8_t *row, int64_t t0, int n) {
  uint32_t bits = 0;
  if (row != nullptr) {
    const int lane = threadIdx.x & 31;
    bits = __ballot_sync(0xffffffffu, lane < n && __ldg(row + t0 + lane) != 0);
  }
  return bits;
}

template <typename T, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 2) recurrence_forward_kernel(const RecurrenceArgs g) {
  __shared__ float2 run_p[2][kWarps][32], run_h[2][kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t batch = blockIdx.x / g.channel_blocks;
  const int64_t ch = int64_t(blockIdx.x % g.channel_blocks) * kChan + first_channel<PAIRED>(lane);
  const bool on0 = ch < g.dim, on1 = ch + kSecond<PAIRED> < g.dim;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + ch;
  const T *value = static_cast<const T *>(g.value) + batch * g.value_batch + ch;
  T *out = static_cast<T *>(g.h) + batch * g.steps * g.dim + ch;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;

  float2 state = make_float2(0.f, 0.f);  // the state before the tile, the same in every warp
  if (g.h0 != nullptr) {
    const float *p = g.h0 + batch * g.dim + ch;
    if (on0) state.x = p[0];
    if (on1) state.y = p[kSecond<PAIRED>];
  }

  int buf = 0;
  for (int64_t tile = 0; tile < g.steps; tile += kTileFwd, buf ^= 1) {
    const int64_t t0 = tile + warp * kRunFwd;
    const int n = static_cast<int>(t0 >= g.steps ? 0 : min64(kRunFwd, g.steps - t0));
    Raw<T> rf[kRunFwd], rx[kRunFwd];
#pragma unroll
    for (int j = 0; j < kRunFwd; ++j) {
      const bool in = j < n;
      rf[j] = load_raw<T, PAIRED>(gate + (t0 + j) * g.gate_step, in && on0, in && on1);
      rx[j] = load_raw<T, PAIRED>(value + (t0 + j) * g.value_step, in && on0, in && on1);
    }
    const uint32_t cut = reset_bits(reset, t0, n);
    const float2 zero = make_float2(0.f, 0.f);
    float2 h = zero, p = make_float2(1.f, 1.f);
    float2 a[kRunFwd], b[kRunFwd];
#pragma unroll
    for (int j = 0; j < kRunFwd; ++j) {
      const float2 f = unpack<T>(rf[j]), x = unpack<T>(rx[j]);
      float2 c;
      gates(f.x, a[j].x, c.x);
      gates(f.y, a[j].y, c.y);
      b[j] = mul2(c, x);
      if (j < n) {
        if ((cut >> j) & 1u) h = p = zero;
        h = fma2(a[j], h, b[j]);
        p = mul2(p, a[j]);
      }
    }
    run_p[buf][warp][lane] = p;
    run_h[buf][warp][lane] = h;
    __syncthreads();
    // The state before this warp's run, and before the next tile.
    float2 in = state;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) in = state;
      const float2 pw = run_p[buf][w][lane], hw = run_h[buf][w][lane];
      state = apply_run(pw, state, hw);
    }
    if (g.saved != nullptr && (warp * kRunFwd) % kTileBwd == 0 && n > 0) {
      float *s = g.saved + (batch * g.saved_tiles + t0 / kTileBwd) * g.dim + ch;
      if (on0) s[0] = in.x;
      if (on1) s[kSecond<PAIRED>] = in.y;
    }
#pragma unroll
    for (int j = 0; j < kRunFwd; ++j) {
      if (j < n) {
        if ((cut >> j) & 1u) in = zero;
        in = fma2(a[j], in, b[j]);
        store_pair<T, PAIRED>(out + (t0 + j) * g.dim, in, on0, on1);
      }
    }
  }
  if (warp == 0) {
    float *p = g.h_last + batch * g.dim + ch;
    if (on0) p[0] = state.x;
    if (on1) p[kSecond<PAIRED>] = state.y;
  }
}

// Backward. With r_t = keep_t a_t ds_t the part of step t's gradient that reaches h_{t-1}:
//   ds_t = grad_t + r_{t+1},  grad_value = c ds,  grad_gate = a c (keep h_{t-1} - x) ds
// h_{t-1} is scanned again from the state saved before the tile (in 32 bits; h itself is not
// read), the same way as forward, and ds the same way from the tile's end: both exchanges of run
// maps share one barrier, and both have the same P.
template <typename T, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 2) recurrence_backward_kernel(const RecurrenceArgs g) {
  __shared__ float2 run_p[2][kWarps][32], run_h[2][kWarps][32], run_r[2][kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t batch = blockIdx.x / g.channel_blocks;
  const int64_t ch = int64_t(blockIdx.x % g.channel_blocks) * kChan + first_channel<PAIRED>(lane);
  const bool on0 = ch < g.dim, on1 = ch + kSecond<PAIRED> < g.dim;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + ch;
  const T *value = static_cast<const T *>(g.value) + batch * g.value_batch + ch;
  const T *grad = g.grad != nullptr ? static_cast<const T *>(g.grad) + batch * g.steps * g.dim + ch : nullptr;
  T *grad_gate = static_cast<T *>(g.grad_gate) + batch * g.steps * g.dim + ch;
  T *grad_value = static_cast<T *>(g.grad_value) + batch * g.steps * g.dim + ch;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;

  float2 back = make_float2(0.f, 0.f);  // r of the step after the tile
  if (g.grad_last != nullptr) {
    const float *p = g.grad_last + batch * g.dim + ch;
    if (on0) back.x = p[0];
    if (on1) back.y = p[kSecond<PAIRED>];
  }

  int buf = 0;
  for (int64_t k = g.saved_tiles - 1; k >= 0; --k, buf ^= 1) {
    const int64_t t0 = k * kTileBwd + warp * kRunBwd;
    const int n = static_cast<int>(t0 >= g.steps ? 0 : min64(kRunBwd, g.steps - t0));
    Raw<T> rf[kRunBwd], rx[kRunBwd], rg[kRunBwd];
#pragma unroll
    for (int j = 0; j < kRunBwd; ++j) {
      const bool in = j < n;
      rf[j] = load_raw<T, PAIRED>(gate + (t0 + j) * g.gate_step, in && on0, in && on1);
      rx[j] = load_raw<T, PAIRED>(value + (t0 + j) * g.value_step, in && on0, in && on1);
      rg[j] = load_raw<T, PAIRED>(grad + (t0 + j) * g.dim, in && on0 && grad != nullptr, in && on1 && grad != nullptr);
    }
    float2 before = make_float2(0.f, 0.f);
    {
      const float *p = g.saved + (batch * g.saved_tiles + k) * g.dim + ch;
      if (on0) before.x = __ldg(p);
      if (on1) before.y = __ldg(p + kSecond<PAIRED>);
    }
    const uint32_t cut = reset_bits(reset, t0, n);

    const float2 zero = make_float2(0.f, 0.f);
    float2 h = zero, p = make_float2(1.f, 1.f), r = zero;
    float2 a[kRunBwd], c[kRunBwd];
#pragma unroll
    for (int j = 0; j < kRunBwd; ++j) {
      const float2 f = unpack<T>(rf[j]), x = unpack<T>(rx[j]);
      gates(f.x, a[j].x, c[j].x);
      gates(f.y, a[j].y, c[j].y);
      if (j < n) {
        if ((cut >> j) & 1u) h = p = zero;
        h = fma2(a[j], h, mul2(c[j], x));
        p = mul2(p, a[j]);
      }
    }
#pragma unroll
    for (int j = kRunBwd - 1; j >= 0; --j) {
      if (j < n) {
        const float2 gt = unpack<T>(rg[j]);
        r = mul2(a[j], make_float2(gt.x + r.x, gt.y + r.y));
        if ((cut >> j) & 1u) r = zero;
      }
    }
    run_p[buf][warp][lane] = p;
    run_h[buf][warp][lane] = h;
    run_r[buf][warp][lane] = r;
    __syncthreads();
    float2 h_in = before, r_in = back;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        const float2 pw = run_p[buf][w][lane], hw = run_h[buf][w][lane];
        h_in = apply_run(pw, h_in, hw);
      }
    }
#pragma unroll
    for (int w = kWarps - 1; w >= 0; --w) {
      if (w == warp) r_in = back;
      const float2 pw = run_p[buf][w][lane], rw = run_r[buf][w][lane];
      back = apply_run(pw, back, rw);
    }
    float2 u[kRunBwd];  // keep h_{t-1} - x
#pragma unroll
    for (int j = 0; j < kRunBwd; ++j) {
      if (j < n) {
        const float2 x = unpack<T>(rx[j]);
        if ((cut >> j) & 1u) h_in = zero;
        u[j] = make_float2(h_in.x - x.x, h_in.y - x.y);
        h_in = fma2(a[j], h_in, mul2(c[j], x));
      }
    }
#pragma unroll
    for (int j = kRunBwd - 1; j >= 0; --j) {
      if (j < n) {
        const float2 gt = unpack<T>(rg[j]);
        const float2 ds = make_float2(gt.x + r_in.x, gt.y + r_in.y);
        const float2 gx = mul2(c[j], ds);
        r_in = mul2(a[j], ds);
        store_pair<T, PAIRED>(grad_value + (t0 + j) * g.dim, gx, on0, on1);
        store_pair<T, PAIRED>(grad_gate + (t0 + j) * g.dim, mul2(mul2(a[j], gx), u[j]), on0, on1);
        if ((cut >> j) & 1u) r_in = zero;
      }
    }
  }
  if (warp == 0 && g.grad_h0 != nullptr) {
    float *p = g.grad_h0 + batch * g.dim + ch;
    if (on0) p[0] = back.x;
    if (on1) p[kSecond<PAIRED>] = back.y;
  }
}

// One token of every row: state (f32, updated in place) and h. A few KB to a few MB: launch
// latency, then one read and one write of each operand.
template <typename T>
__global__ void __launch_bounds__(256) recurrence_step_kernel(const T *__restrict__ gate, int64_t gate_row,
                                                              const T *__restrict__ value, int64_t value_row,
                                                              const uint8_t *__restrict__ reset, int64_t dim,
                                                              float *state, int64_t state_row, T *__restrict__ h) {
  const int64_t ch = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = blockIdx.y;
  if (ch >= dim) return;
  const float before = reset != nullptr && reset[row] != 0 ? 0.f : state[row * state_row + ch];
  float a, c;
  gates(to_f32<T>(gate[row * gate_row + ch]), a, c);
  const float now = fmaf(a, before, c * to_f32<T>(value[row * value_row + ch]));
  state[row * state_row + ch] = now;
  h[row * dim + ch] = from_f32<T>(now);
}

inline size_t elem_bytes(int dtype) { return dtype == TROPNN_B200_F32 ? 4 : 2; }
inline bool paired(const void *p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (2 * elem_bytes(dtype)) == 0; }

int check_sizes(const char *what, int dtype, int64_t batch, int64_t steps, int64_t dim) {
  TB_REQUIRE(is_float_dtype(dtype), TROPNN_B200_ERR_DTYPE, "%s: dtype %d is not f32/f16/bf16", what, dtype);
  TB_REQUIRE(batch >= 0 && steps >= 0 && dim >= 0, TROPNN_B200_ERR_INVALID, "%s: bad sizes (batch %lld, steps %lld, dim %lld)",
             what, (long long)batch, (long long)steps, (long long)dim);
  TB_REQUIRE(batch * ceil_div(dim, kChan) <= 0x7fffffffLL, TROPNN_B200_ERR_INVALID, "%s: batch x dim too large", what);
  return TROPNN_B200_OK;
}

template <bool BACKWARD>
int launch_recurrence(const char *what, const RecurrenceArgs &g, int dtype, int64_t batch, bool pair, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(batch * g.channel_blocks);
#define TB_LAUNCH(T, PAIR)                                                                  \
  do {                                                                                      \
    if (BACKWARD)                                                                           \
      recurrence_backward_kernel<T, PAIR><<<grid, kThreads, 0, stream>>>(g);                \
    else                                                                                    \
      recurrence_forward_kernel<T, PAIR><<<grid, kThreads, 0, stream>>>(g);                 \
  } while (0)
  if (dtype == TROPNN_B200_F32) {
    if (pair) TB_LAUNCH(float, true); else TB_LAUNCH(float, false);
  } else if (dtype == TROPNN_B200_F16) {
    if (pair) TB_LAUNCH(__half, true); else TB_LAUNCH(__half, false);
  } else {
    if (pair) TB_LAUNCH(__nv_bfloat16, true); else TB_LAUNCH(__nv_bfloat16, false);
  }
#undef TB_LAUNCH
  return check_launch(what);
}

}  // namespace
}  // namespace tropnn_b200

using namespace tropnn_b200;

extern "C" {

size_t tropnn_b200_recurrence_saved_size(int64_t batch, int64_t steps, int64_t dim) {
  if (batch <= 0 || steps <= 0 || dim <= 0) return 0;
  return static_cast<size_t>(batch * ceil_div(steps, kTileBwd) * dim) * sizeof(float);
}

int tropnn_b200_recurrence_forward(const void *gate, int64_t gate_batch_stride, int64_t gate_step_stride,
                                   const void *value, int64_t value_batch_stride, int64_t value_step_stride, int dtype,
                                   const float *h0, const uint8_t *reset, int64_t batch, int64_t steps, int64_t dim,
                                   void *h, float *h_last, float *saved, size_t saved_bytes, void *stream) {
  const char *what = "recurrence_forward";
  TB_CHECK(check_sizes(what, dtype, batch, steps, dim));
  if (batch == 0 || dim == 0) return clear_error();
  TB_REQUIRE(h_last != nullptr && (steps == 0 || (gate != nullptr && value != nullptr && h != nullptr)),
             TROPNN_B200_ERR_INVALID, "%s: null pointer", what);
  TB_REQUIRE(saved == nullptr || saved_bytes >= tropnn_b200_recurrence_saved_size(batch, steps, dim),
             TROPNN_B200_ERR_WORKSPACE, "%s: %zu bytes of saved states, %zu needed", what, saved_bytes,
             tropnn_b200_recurrence_saved_size(batch, steps, dim));
  TB_CHECK(check_current_device());
  RecurrenceArgs g{};
  g.gate = gate;
  g.value = value;
  g.gate_batch = gate_batch_stride;
  g.gate_step = gate_step_stride;
  g.value_batch = value_batch_stride;
  g.value_step = value_step_stride;
  g.h0 = h0;
  g.reset = reset;
  g.steps = steps;
  g.dim = dim;
  g.channel_blocks = static_cast<int>(ceil_div(dim, kChan));
  g.h = h;
  g.h_last = h_last;
  g.saved = saved;
  g.saved_tiles = ceil_div(steps, kTileBwd);
  const bool pair = dim % 2 == 0 && gate_batch_stride % 2 == 0 && gate_step_stride % 2 == 0 &&
                    value_batch_stride % 2 == 0 && value_step_stride % 2 == 0 && paired(gate, dtype) &&
                    paired(value, dtype) && paired(h, dtype);
  TB_CHECK((launch_recurrence<false>(what, g, dtype, batch, pair, as_stream(stream))));
  return clear_error();
}

int tropnn_b200_recurrence_backward(const void *gate, int64_t gate_batch_stride, int64_t gate_step_stride,
                                    const void *value, int64_t value_batch_stride, int64_t value_step_stride, int dtype,
                                    const uint8_t *reset, int64_t batch, int64_t steps, int64_t dim, const float *saved,
                                    size_t saved_bytes, const void *grad, const float *grad_last, void *grad_gate,
                                    void *grad_value, float *grad_h0, void *stream) {
  const char *what = "recurrence_backward";
  TB_CHECK(check_sizes(what, dtype, batch, steps, dim));
  if (batch == 0 || dim == 0) return clear_error();
  TB_REQUIRE(steps == 0 || (gate != nullptr && value != nullptr && saved != nullptr && grad_gate != nullptr && grad_value != nullptr),
             TROPNN_B200_ERR_INVALID, "%s: null pointer", what);
  TB_REQUIRE(saved_bytes >= tropnn_b200_recurrence_saved_size(batch, steps, dim), TROPNN_B200_ERR_WORKSPACE,
             "%s: %zu bytes of saved states, %zu needed", what, saved_bytes,
             tropnn_b200_recurrence_saved_size(batch, steps, dim));
  TB_CHECK(check_current_device());
  RecurrenceArgs g{};
  g.gate = gate;
  g.value = value;
  g.gate_batch = gate_batch_stride;
  g.gate_step = gate_step_stride;
  g.value_batch = value_batch_stride;
  g.value_step = value_step_stride;
  g.reset = reset;
  g.steps = steps;
  g.dim = dim;
  g.channel_blocks = static_cast<int>(ceil_div(dim, kChan));
  g.saved = const_cast<float *>(saved);
  g.saved_tiles = ceil_div(steps, kTileBwd);
  g.grad = grad;
  g.grad_last = grad_last;
  g.grad_gate = grad_gate;
  g.grad_value = grad_value;
  g.grad_h0 = grad_h0;
  const bool pair = dim % 2 == 0 && gate_batch_stride % 2 == 0 && gate_step_stride % 2 == 0 &&
                    value_batch_stride % 2 == 0 && value_step_stride % 2 == 0 && paired(gate, dtype) &&
                    paired(value, dtype) && paired(grad, dtype) && paired(grad_gate, dtype) && paired(grad_value, dtype);
  TB_CHECK((launch_recurrence<true>(what, g, dtype, batch, pair, as_stream(stream))));
  return clear_error();
}

int tropnn_b200_recurrence_step(const void *gate, int64_t gate_stride, const void *value, int64_t value_stride,
                                int dtype, const uint8_t *reset, int64_t batch, int64_t dim, float *state,
                                int64_t state_stride, void *h, void *stream) {
  const char *what = "recurrence_step";
  TB_CHECK(check_sizes(what, dtype, batch, 1, dim));
  if (batch == 0 || dim == 0) return clear_error();
  TB_REQUIRE(gate != nullptr && value != nullptr && state != nullptr && h != nullptr, TROPNN_B200_ERR_INVALID,
             "%s: null pointer", what);
  TB_CHECK(check_current_device());
  int64_t done = 0;
  while (done < batch) {  // a launch takes 65535 rows (the grid's y extent)
    const int64_t rows = min64(batch - done, 65535);
    const dim3 grid(static_cast<unsigned>(ceil_div(dim, 256)), static_cast<unsigned>(rows));
    const size_t eb = elem_bytes(dtype);
    const char *gp = static_cast<const char *>(gate) + done * gate_stride * int64_t(eb);
    const char *vp = static_cast<const char *>(value) + done * value_stride * int64_t(eb);
    char *hp = static_cast<char *>(h) + done * dim * int64_t(eb);
    const uint8_t *rp = reset != nullptr ? reset + done : nullptr;
    float *sp = state + done * state_stride;
#define TB_STEP(T)                                                                                              \
  recurrence_step_kernel<T><<<grid, 256, 0, as_stream(stream)>>>(reinterpret_cast<const T *>(gp), gate_stride,   \
                                                                 reinterpret_cast<const T *>(vp), value_stride, rp, \
                                                                 dim, sp, state_stride, reinterpret_cast<T *>(hp))
    if (dtype == TROPNN_B200_F32) TB_STEP(float);
    else if (dtype == TROPNN_B200_F16) TB_STEP(__half);
    else TB_STEP(__nv_bfloat16);
#undef TB_STEP
    TB_CHECK(check_launch(what));
    done += rows;
  }
  return clear_error();
}

}  // extern "C"
