// Gated linear recurrence over token sequences: forward, backward and the single-token step.
//
//   a_t = sigmoid(f_t), c_t = 1 - a_t = sigmoid(-f_t)          (per channel)
//   h_t = keep_t a_t h_{t-1} + c_t x_t                          (keep_t = 0 at a reset, else 1)
//
// The recurrence is linear, so a run of steps maps the state before it to P h + H with P the
// product of its keep_t a_t. A warp owns a run of consecutive steps of 64 channels (two a lane): it
// scans them in registers from h = 0 for (P, H), hands those to the other warps through shared
// memory, composes the runs before its own into its incoming state and scans again from there.
// A CTA's 8 warps take a tile of 8 runs. One read of gate and value, one write of h: the kernels are
// bound by HBM traffic where enough CTAs are at work:
//  - a cluster of up to 8 CTAs takes as many consecutive tiles at once and exchanges their maps
//    through distributed shared memory, while the next tiles' loads are under way;
//  - with too few channels for that (a long sequence of a small batch) the sequence is cut into
//    chunks: a first launch computes each chunk's map, and every chunk composes those before its own.
//    The inputs are then read twice, the second time largely from L2.
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChan = 64;                    // channels of a CTA, two a lane
// Steps of a warp's run: what leaves room for the next tile's values in 128 registers a thread.
template <typename T>
constexpr int kRunFwd = sizeof(T) == 2 ? 16 : 8;
constexpr int kRunBwd = 8;
constexpr int kTileBwd = kWarps * kRunBwd;  // 64: also the distance of the saved states
static_assert(kTileBwd % kRunFwd<float> == 0 && kTileBwd % kRunFwd<__half> == 0, "saved states start at a run");
constexpr int kMaxCluster = 8;
constexpr int kSlots = 2 * 148;  // CTAs at once

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

// `second`: distance of the lane's second channel (PAIRED: 1).
template <typename T, bool PAIRED>
__device__ __forceinline__ Raw<T> load_raw(const T *p, int second) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    if constexpr (PAIRED) {
      const float2 q = __ldg(reinterpret_cast<const float2 *>(p));
      r.a = q.x;
      r.b = q.y;
    } else {
      r.a = __ldg(p);
      r.b = __ldg(p + second);
    }
  } else {
    if constexpr (PAIRED) {
      r.v = __ldg(reinterpret_cast<const unsigned int *>(p));
    } else {
      const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
      r.v = uint32_t(__ldg(u)) | (uint32_t(__ldg(u + second)) << 16);
    }
  }
  return r;
}

// A lane's two channels: where it stores, and where it loads. Lanes past the last channel load
// channels that are there and store nothing.
template <bool PAIRED>
struct Lane {
  int64_t ch;      // first channel
  bool on0, on1;   // which of the two are there
  int64_t from;    // loads: first channel, and the second's distance
  int second;
  __device__ __forceinline__ Lane(int64_t block, int64_t dim) {
    const int lane = threadIdx.x & 31;
    ch = block * kChan + first_channel<PAIRED>(lane);
    on0 = ch < dim;
    on1 = ch + kSecond<PAIRED> < dim;
    from = on0 ? ch : (PAIRED ? dim - 2 : dim - 1);
    second = PAIRED ? 1 : (on1 ? 32 : 0);
  }
};

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
    if constexpr (PAIRED) {
      uint32_t w;
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 q = __float22half2_rn(v);
        w = *reinterpret_cast<const uint32_t *>(&q);
      } else {
        const __nv_bfloat162 q = __float22bfloat162_rn(v);
        w = *reinterpret_cast<const uint32_t *>(&q);
      }
      if (on0) *reinterpret_cast<uint32_t *>(p) = w;
    } else {
      if (on0) p[0] = from_f32<T>(v.x);
      if (on1) p[32] = from_f32<T>(v.y);
    }
  }
}

// a and c = 1 - a. The smaller one, m = e / (1 + e) with e = exp(-|f|), has its full relative
// accuracy; the larger is 1 - m, the f32 next to it.
__device__ __forceinline__ void gates1(float f, float &a, float &c) {
  const float e = exp2_approx(fabsf(f) * -1.4426950408889634f);
  const float m = e * rcp_approx(1.f + e), o = 1.f - m;
  a = f < 0.f ? m : o;
  c = f < 0.f ? o : m;
}
__device__ __forceinline__ void gates2(float2 f, float2 &a, float2 &c) {
  gates1(f.x, a.x, c.x);
  gates1(f.y, a.y, c.y);
}

// P h + H. With resets about (`cuts`), a run that one cut (P = 0) takes nothing of h, not even an
// infinity's NaN.
__device__ __forceinline__ float2 apply_run(float2 p, float2 h, float2 add, bool cuts) {
  if (!cuts) return fma2(p, h, add);
  return make_float2(p.x == 0.f ? add.x : fmaf(p.x, h.x, add.x), p.y == 0.f ? add.y : fmaf(p.y, h.y, add.y));
}

struct RecurrenceArgs {
  const void *gate, *value;
  int64_t gate_batch, gate_step, value_batch, value_step;
  const float *h0;
  const uint8_t *reset;
  int64_t steps, dim;
  int channel_blocks;
  int ranks;            // CTAs of a cluster
  int chunks;           // of the sequence, each a launch-grid row
  int64_t chunk_tiles;  // tiles of a chunk
  float2 *maps;         // chunks > 1: (P, H) or (P, R) of [batch, chunk, dim]
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Exchange of run maps: (P, H) of the CTA's warps and of the cluster's CTAs, two lane channels each.
struct Exchange {
  float2 p[2][kWarps][32], h[2][kWarps][32];
  float4 rank[2][kMaxCluster][32];
};

// The chunks' maps before (FORWARD) or after this one, composed onto `state`: the warps take a share
// each, in order.
template <bool PAIRED, bool FORWARD>
__device__ __forceinline__ float2 through_chunks(const RecurrenceArgs &g, int64_t batch, int64_t ch, bool on0, bool on1,
                                                 int chunk, float2 state, Exchange &ex) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = FORWARD ? chunk : g.chunks - 1 - chunk;
  const int share = (count + kWarps - 1) / kWarps;
  const int first = min(warp * share, count), stop = min(first + share, count);
  float2 p = make_float2(1.f, 1.f), h = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int i = first; i < stop; ++i) {
    const int q = FORWARD ? i : g.chunks - 1 - i;
    const float2 *m = g.maps + (batch * g.chunks + q) * g.dim + ch;
    float2 a = make_float2(1.f, 0.f), b = make_float2(1.f, 0.f);
    if (on0) a = __ldg(m);
    if (on1) b = __ldg(m + kSecond<PAIRED>);
    const float2 mp = make_float2(a.x, b.x);
    h = apply_run(mp, h, make_float2(a.y, b.y), true);
    p = mul2(mp, p);
  }
  ex.p[0][warp][lane] = p;
  ex.h[0][warp][lane] = h;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) state = apply_run(ex.p[0][w][lane], state, ex.h[0][w][lane], true);
  __syncthreads();
  return state;
}

// Hands this warp's (p, h) around: returns the state before its run, and moves `state` past the
// cluster's tiles. ORDER 1: the runs follow one another by warp, -1: from the last warp back.
template <int ORDER>
__device__ __forceinline__ float2 exchange(Exchange &ex, int buf, float2 p, float2 h, float2 &state, int ranks, int rank,
                                           bool cuts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ex.p[buf][warp][lane] = p;
  ex.h[buf][warp][lane] = h;
  __syncthreads();
  float2 in = state;
  if (ranks == 1) {
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int w = ORDER > 0 ? i : kWarps - 1 - i;
      if (w == warp) in = state;
      state = apply_run(ex.p[buf][w][lane], state, ex.h[buf][w][lane], cuts);
    }
    return in;
  }
  if (warp < ranks) {  // the CTA's map, to one CTA a warp
    float2 cp = make_float2(1.f, 1.f), ch = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int w = ORDER > 0 ? i : kWarps - 1 - i;
      const float2 pw = ex.p[buf][w][lane];
      ch = apply_run(pw, ch, ex.h[buf][w][lane], cuts);
      cp = mul2(cp, pw);
    }
    *cooperative_groups::this_cluster().map_shared_rank(&ex.rank[buf][rank][lane], warp) = make_float4(cp.x, cp.y, ch.x, ch.y);
  }
  cluster_arrive();
  cluster_wait();
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) in = state;
    const float4 m = ex.rank[buf][r][lane];
    state = apply_run(make_float2(m.x, m.y), state, make_float2(m.z, m.w), cuts);
  }
#pragma unroll
  for (int i = 0; i < kWarps - 1; ++i) {
    const int w = ORDER > 0 ? i : kWarps - 1 - i;
    if (ORDER > 0 ? w < warp : w > warp) in = apply_run(ex.p[buf][w][lane], in, ex.h[buf][w][lane], cuts);
  }
  return in;
}

// The reset flags of `n` consecutive steps as bits.
__device__ __forceinline__ uint32_t reset_bits(const uint8_t *row, int64_t t0, int n) {
  uint32_t bits = 0;
  if (row != nullptr) {
    const int lane = threadIdx.x & 31;
    bits = __ballot_sync(0xffffffffu, lane < n && __ldg(row + t0 + lane) != 0);
  }
  return bits;
}

// A run's map from its gates and c x: (p, h). `plain`: all its steps are there and none is a reset.
template <int RUN>
__device__ __forceinline__ void scan_run(const float2 (&a)[RUN], const float2 (&b)[RUN], int n, uint32_t cut, bool plain,
                                         float2 &p, float2 &h) {
  const float2 zero = make_float2(0.f, 0.f);
  h = zero;
  p = make_float2(1.f, 1.f);
  if (plain) {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      h = fma2(a[j], h, b[j]);
      p = mul2(p, a[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j < n) {
        if ((cut >> j) & 1u) h = p = zero;
        h = fma2(a[j], h, b[j]);
        p = mul2(p, a[j]);
      }
    }
  }
}
// The run from the state before it: store(j, h_j).
template <int RUN, typename Store>
__device__ __forceinline__ void emit_run(const float2 (&a)[RUN], const float2 (&b)[RUN], int n, uint32_t cut, bool plain,
                                         float2 in, Store store) {
  if (plain) {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      in = fma2(a[j], in, b[j]);
      store(j, in);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j < n) {
        if ((cut >> j) & 1u) in = make_float2(0.f, 0.f);
        in = fma2(a[j], in, b[j]);
        store(j, in);
      }
    }
  }
}
// Backward: a run's maps, (p, h) forward and (p, r) from its end.
template <int RUN>
__device__ __forceinline__ void scan_run_back(const float2 (&a)[RUN], const float2 (&c)[RUN], const float2 (&x)[RUN],
                                              const float2 (&gt)[RUN], int n, uint32_t cut, bool plain, float2 &p,
                                              float2 &h, float2 &r) {
  const float2 zero = make_float2(0.f, 0.f);
  h = r = zero;
  p = make_float2(1.f, 1.f);
  if (plain) {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      h = fma2(a[j], h, mul2(c[j], x[j]));
      p = mul2(p, a[j]);
    }
#pragma unroll
    for (int j = RUN - 1; j >= 0; --j) r = mul2(a[j], add2(gt[j], r));
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j < n) {
        if ((cut >> j) & 1u) h = p = zero;
        h = fma2(a[j], h, mul2(c[j], x[j]));
        p = mul2(p, a[j]);
      }
    }
#pragma unroll
    for (int j = RUN - 1; j >= 0; --j) {
      if (j < n) {
        r = mul2(a[j], add2(gt[j], r));
        if ((cut >> j) & 1u) r = zero;
      }
    }
  }
}
// The run's gradients from the state before it and r after it: store(j, grad_gate, grad_value), from
// the last step back. x is used up.
template <int RUN, typename Store>
__device__ __forceinline__ void emit_run_back(const float2 (&a)[RUN], const float2 (&c)[RUN], float2 (&x)[RUN],
                                              const float2 (&gt)[RUN], int n, uint32_t cut, bool plain, float2 h_in,
                                              float2 r_in, Store store) {
  const float2 zero = make_float2(0.f, 0.f), minus = make_float2(-1.f, -1.f);
  if (plain) {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      const float2 v = x[j];
      x[j] = fma2(v, minus, h_in);  // keep h_{t-1} - x
      h_in = fma2(a[j], h_in, mul2(c[j], v));
    }
#pragma unroll
    for (int j = RUN - 1; j >= 0; --j) {
      const float2 ds = add2(gt[j], r_in), gx = mul2(c[j], ds);
      r_in = mul2(a[j], ds);
      store(j, mul2(mul2(a[j], gx), x[j]), gx);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j < n) {
        const float2 v = x[j];
        if ((cut >> j) & 1u) h_in = zero;
        x[j] = fma2(v, minus, h_in);
        h_in = fma2(a[j], h_in, mul2(c[j], v));
      }
    }
#pragma unroll
    for (int j = RUN - 1; j >= 0; --j) {
      if (j < n) {
        const float2 ds = add2(gt[j], r_in), gx = mul2(c[j], ds);
        r_in = mul2(a[j], ds);
        store(j, mul2(mul2(a[j], gx), x[j]), gx);
        if ((cut >> j) & 1u) r_in = zero;
      }
    }
  }
}

template <typename T, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 2) recurrence_forward_kernel(const RecurrenceArgs g) {
  constexpr int kRun = kRunFwd<T>, kTile = kWarps * kRun;
  __shared__ Exchange ex;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % g.ranks, chunk = blockIdx.y;
  const int unit = blockIdx.x / g.ranks;
  const int64_t batch = unit / g.channel_blocks;
  const Lane<PAIRED> at(unit % g.channel_blocks, g.dim);
  const int64_t ch = at.ch;
  const bool on0 = at.on0, on1 = at.on1;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
  const T *value = static_cast<const T *>(g.value) + batch * g.value_batch + at.from;
  T *out = static_cast<T *>(g.h) + batch * g.steps * g.dim + ch;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t first = chunk * g.chunk_tiles * kTile, stop = min64(g.steps, first + g.chunk_tiles * kTile);
  if (g.ranks > 1) cluster_arrive();

  Raw<T> rf[kRun], rx[kRun];
  auto load = [&](int64_t t0) {
    if (t0 >= stop) return;
    // Steps past the end load the last one again.
    const int64_t most = stop - 1 - t0;
    const T *pf = gate + t0 * g.gate_step, *px = value + t0 * g.value_step;
    if (most >= kRun - 1) {
#pragma unroll
      for (int j = 0; j < kRun; ++j, pf += g.gate_step, px += g.value_step) {
        rf[j] = load_raw<T, PAIRED>(pf, at.second);
        rx[j] = load_raw<T, PAIRED>(px, at.second);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        rf[j] = load_raw<T, PAIRED>(pf + min64(j, most) * g.gate_step, at.second);
        rx[j] = load_raw<T, PAIRED>(px + min64(j, most) * g.value_step, at.second);
      }
    }
  };
  load(first + rank * kTile + warp * kRun);
  float2 state = make_float2(0.f, 0.f);  // the state before the cluster's tiles, the same in every warp
  if (g.h0 != nullptr) {
    const float *p = g.h0 + batch * g.dim + ch;
    if (on0) state.x = p[0];
    if (on1) state.y = p[kSecond<PAIRED>];
  }
  if (chunk > 0) state = through_chunks<PAIRED, true>(g, batch, ch, on0, on1, chunk, state, ex);
  if (g.ranks > 1) cluster_wait();

  int buf = 0;
  for (int64_t tile = first; tile < stop; tile += int64_t(g.ranks) * kTile, buf ^= 1) {
    const int64_t t0 = tile + rank * kTile + warp * kRun;
    const int n = static_cast<int>(t0 >= stop ? 0 : min64(kRun, stop - t0));
    const uint32_t cut = reset_bits(reset, t0, n);
    const bool plain = n == kRun && cut == 0;
    float2 a[kRun], b[kRun], p, h;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      float2 c;
      gates2(unpack<T>(rf[j]), a[j], c);
      b[j] = mul2(c, unpack<T>(rx[j]));
    }
    scan_run<kRun>(a, b, n, cut, plain, p, h);
    load(t0 + int64_t(g.ranks) * kTile);
    const float2 in = exchange<1>(ex, buf, p, h, state, g.ranks, rank, reset != nullptr);
    if (g.saved != nullptr && (warp * kRun) % kTileBwd == 0 && n > 0) {
      float *s = g.saved + (batch * g.saved_tiles + t0 / kTileBwd) * g.dim + ch;
      if (on0) s[0] = in.x;
      if (on1) s[kSecond<PAIRED>] = in.y;
    }
    T *po = out + t0 * g.dim;
    emit_run<kRun>(a, b, n, cut, plain, in, [&](int, float2 v) {
      store_pair<T, PAIRED>(po, v, on0, on1);
      po += g.dim;
    });
  }
  if (warp == 0 && rank == 0 && chunk == g.chunks - 1) {
    float *p = g.h_last + batch * g.dim + ch;
    if (on0) p[0] = state.x;
    if (on1) p[kSecond<PAIRED>] = state.y;
  }
}

// Backward. With r_t = keep_t a_t ds_t the part of step t's gradient that reaches h_{t-1}:
//   ds_t = grad_t + r_{t+1},  grad_value = c ds,  grad_gate = a c (keep h_{t-1} - x) ds
// h_{t-1} is scanned again from the state saved before the tile (in 32 bits; h itself is not
// read), the same way as forward within the tile; r comes from the sequence's end, across the
// cluster's tiles. Both have the same P.
template <typename T, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 2) recurrence_backward_kernel(const RecurrenceArgs g) {
  constexpr int kRun = kRunBwd, kTile = kTileBwd;
  __shared__ Exchange ex;
  __shared__ float2 run_h[2][kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % g.ranks, chunk = blockIdx.y;
  const int unit = blockIdx.x / g.ranks;
  const int64_t batch = unit / g.channel_blocks;
  const Lane<PAIRED> at(unit % g.channel_blocks, g.dim);
  const int64_t ch = at.ch;
  const bool on0 = at.on0, on1 = at.on1;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
  const T *value = static_cast<const T *>(g.value) + batch * g.value_batch + at.from;
  const T *grad = g.grad != nullptr ? static_cast<const T *>(g.grad) + batch * g.steps * g.dim + at.from : nullptr;
  T *grad_gate = static_cast<T *>(g.grad_gate) + batch * g.steps * g.dim + ch;
  T *grad_value = static_cast<T *>(g.grad_value) + batch * g.steps * g.dim + ch;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t first = chunk * g.chunk_tiles, stop = min64(g.saved_tiles, first + g.chunk_tiles);
  if (g.ranks > 1) cluster_arrive();

  Raw<T> rf[kRun], rx[kRun], rg[kRun] = {};
  float2 before = make_float2(0.f, 0.f);
  auto steps_of = [&](int64_t k) -> int {
    const int64_t t0 = k * kTile + warp * kRun;
    return static_cast<int>(k < first || t0 >= g.steps ? 0 : min64(kRun, g.steps - t0));
  };
  auto load = [&](int64_t k) {
    if (k < first) return;
    // Steps past the end load the last one again.
    const int64_t t0 = k * kTile + warp * kRun, from = min64(t0, g.steps - 1), most = g.steps - 1 - from;
    const T *pf = gate + from * g.gate_step, *px = value + from * g.value_step, *pg = grad + from * g.dim;
    if (most >= kRun - 1) {
#pragma unroll
      for (int j = 0; j < kRun; ++j, pf += g.gate_step, px += g.value_step, pg += g.dim) {
        rf[j] = load_raw<T, PAIRED>(pf, at.second);
        rx[j] = load_raw<T, PAIRED>(px, at.second);
        if (grad != nullptr) rg[j] = load_raw<T, PAIRED>(pg, at.second);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int64_t d = min64(j, most);
        rf[j] = load_raw<T, PAIRED>(pf + d * g.gate_step, at.second);
        rx[j] = load_raw<T, PAIRED>(px + d * g.value_step, at.second);
        if (grad != nullptr) rg[j] = load_raw<T, PAIRED>(pg + d * g.dim, at.second);
      }
    }
    const float *p = g.saved + (batch * g.saved_tiles + k) * g.dim + at.from;
    before = make_float2(__ldg(p), __ldg(p + at.second));
  };
  load(stop - 1 - rank);
  float2 back = make_float2(0.f, 0.f);  // r of the step after the cluster's tiles
  if (g.grad_last != nullptr) {
    const float *p = g.grad_last + batch * g.dim + ch;
    if (on0) back.x = p[0];
    if (on1) back.y = p[kSecond<PAIRED>];
  }
  if (chunk < g.chunks - 1) back = through_chunks<PAIRED, false>(g, batch, ch, on0, on1, chunk, back, ex);
  if (g.ranks > 1) cluster_wait();

  int buf = 0;
  for (int64_t last = stop - 1; last >= first; last -= g.ranks, buf ^= 1) {
    const int64_t k = last - rank, t0 = k * kTile + warp * kRun;
    const int n = steps_of(k);
    const uint32_t cut = reset_bits(reset, t0, n);

    const bool plain = n == kRun && cut == 0;
    float2 a[kRun], c[kRun], x[kRun], gt[kRun], p, h, r, h_in = before;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      gates2(unpack<T>(rf[j]), a[j], c[j]);
      x[j] = unpack<T>(rx[j]);
      gt[j] = unpack<T>(rg[j]);
    }
    scan_run_back<kRun>(a, c, x, gt, n, cut, plain, p, h, r);
    load(k - g.ranks);
    run_h[buf][warp][lane] = h;
    const float2 r_in = exchange<-1>(ex, buf, p, r, back, g.ranks, rank, reset != nullptr);
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w) {
      if (w < warp) h_in = apply_run(ex.p[buf][w][lane], h_in, run_h[buf][w][lane], reset != nullptr);
    }
    T *pf = grad_gate + t0 * g.dim, *px = grad_value + t0 * g.dim;
    emit_run_back<kRun>(a, c, x, gt, n, cut, plain, h_in, r_in, [&](int j, float2 gf, float2 gx) {
      store_pair<T, PAIRED>(px + j * g.dim, gx, on0, on1);
      store_pair<T, PAIRED>(pf + j * g.dim, gf, on0, on1);
    });
  }
  if (warp == 0 && rank == 0 && chunk == 0 && g.grad_h0 != nullptr) {
    float *p = g.grad_h0 + batch * g.dim + ch;
    if (on0) p[0] = back.x;
    if (on1) p[kSecond<PAIRED>] = back.y;
  }
}

// The same two kernels with the data brought by TMA: each warp has its own ring of stages in shared
// memory, loads its runs of [steps x 64 channels] into them two or three tiles ahead, writes its
// results over the inputs of the stage and stores them from there. No registers hold data in
// flight, no address is computed an element, rows and channels that are not there come as zeros and
// are not written. Needs rows 16 bytes aligned (dim and strides multiples of 8 16-bit or 4 f32
// elements); the kernels above serve all else.
struct SequenceMaps {
  CUtensorMap gate, value, grad, out_gate, out_value;  // out_value: h in the forward
};
__device__ int g_recurrence_error = 0;

__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, const void *src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(sm100::smem_addr(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

template <typename T>
__device__ __forceinline__ Raw<T> stage_raw(const T *row, int lane) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    const float2 q = reinterpret_cast<const float2 *>(row)[lane];
    r.a = q.x;
    r.b = q.y;
  } else {
    r.v = reinterpret_cast<const uint32_t *>(row)[lane];
  }
  return r;
}

// Neighbours in an f32 array that may start anywhere.
__device__ __forceinline__ float2 two_floats(const float *p) { return make_float2(__ldg(p), __ldg(p + 1)); }
__device__ __forceinline__ void put_two_floats(float *p, float2 v) {
  p[0] = v.x;
  p[1] = v.y;
}

template <typename T>
constexpr int kStagesFwd = 3;
template <typename T>
constexpr int kStagesBwd = sizeof(T) == 2 ? 3 : 2;
template <typename T, bool FORWARD>
constexpr size_t kRingBytes = FORWARD ? size_t(kWarps) * kStagesFwd<T> * 2 * kRunFwd<T> * kChan * sizeof(T)
                                      : size_t(kWarps) * kStagesBwd<T> * 3 * kRunBwd * kChan * sizeof(T);

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    recurrence_forward_tma_kernel(const RecurrenceArgs g, const __grid_constant__ SequenceMaps maps) {
  constexpr int kRun = kRunFwd<T>, kTile = kWarps * kRun, kStages = kStagesFwd<T>;
  constexpr uint32_t kBytes = 2 * kRun * kChan * sizeof(T);
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ Exchange ex;
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % g.ranks, chunk = blockIdx.y;
  const int unit = blockIdx.x / g.ranks;
  const int batch = unit / g.channel_blocks, ch0 = unit % g.channel_blocks * kChan;
  const int64_t ch = ch0 + 2 * lane;
  const bool on = ch < g.dim;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t first = chunk * g.chunk_tiles * kTile, stop = min64(g.steps, first + g.chunk_tiles * kTile);
  const int64_t stride = int64_t(g.ranks) * kTile;
  T *ring = reinterpret_cast<T *>(dynamic) + size_t(warp) * kStages * 2 * kRun * kChan;
  auto stage = [&](int s) -> T * { return ring + s * 2 * kRun * kChan; };
  auto fetch = [&](int64_t t0, int s) {  // one lane
    if (t0 >= stop) return;
    sm100::mbar_expect_tx(&full[warp][s], kBytes);
    sm100::tma_load_3d(stage(s), &maps.gate, &full[warp][s], ch0, static_cast<int>(t0), batch);
    sm100::tma_load_3d(stage(s) + kRun * kChan, &maps.value, &full[warp][s], ch0, static_cast<int>(t0), batch);
  };
  auto flag_of = [&](int64_t t0) -> uint32_t {
    return reset != nullptr && lane < kRun && t0 + lane < stop ? __ldg(reset + t0 + lane) : 0u;
  };
  if (g.ranks > 1) cluster_arrive();
  if (threadIdx.x == 0) abort = 0;
  const int64_t t_first = first + rank * kTile + warp * kRun;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) sm100::mbar_init(&full[warp][s], 1);
    sm100::mbar_init_fence();
    sm100::fence_proxy_async_smem();
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(t_first + s * stride, s);
  }
  uint32_t flag = flag_of(t_first);
  __syncthreads();

  float2 state = make_float2(0.f, 0.f);
  if (g.h0 != nullptr && on) state = two_floats(g.h0 + batch * g.dim + ch);
  if (chunk > 0) state = through_chunks<true, true>(g, batch, ch, on, on, chunk, state, ex);
  if (g.ranks > 1) cluster_wait();

  int buf = 0, s = 0;
  uint32_t parity = 0;
  for (int64_t tile = first, t0 = t_first; tile < stop; tile += stride, t0 += stride, buf ^= 1) {
    const int n = static_cast<int>(t0 >= stop ? 0 : min64(kRun, stop - t0));
    const uint32_t cut = __ballot_sync(0xffffffffu, flag != 0);
    flag = flag_of(t0 + stride);
    const bool plain = n == kRun && cut == 0;
    if (n > 0) sm100::mbar_wait(&full[warp][s], parity, &abort, &g_recurrence_error);
    T *rows = stage(s);
    float2 a[kRun], b[kRun], p, h;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      float2 c;
      gates2(unpack<T>(stage_raw<T>(rows + j * kChan, lane)), a[j], c);
      b[j] = mul2(c, unpack<T>(stage_raw<T>(rows + (kRun + j) * kChan, lane)));
    }
    scan_run<kRun>(a, b, n, cut, plain, p, h);
    const float2 in = exchange<1>(ex, buf, p, h, state, g.ranks, rank, reset != nullptr);
    if (g.saved != nullptr && (warp * kRun) % kTileBwd == 0 && n > 0 && on)
      put_two_floats(g.saved + (batch * g.saved_tiles + t0 / kTileBwd) * g.dim + ch, in);
    emit_run<kRun>(a, b, n, cut, plain, in,
                   [&](int j, float2 v) { store_pair<T, true>(rows + (kRun + j) * kChan + 2 * lane, v, true, true); });
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (n > 0) tma_store_3d(&maps.out_value, rows + kRun * kChan, ch0, static_cast<int>(t0), batch);
      sm100::bulk_commit();
      // The stage before this one has been read by its store: its next tile comes in.
      bulk_wait_read<1>();
      if (tile > first) fetch(t0 + (kStages - 1) * stride, s == 0 ? kStages - 1 : s - 1);
    }
    if (++s == kStages) {
      s = 0;
      parity ^= 1;
    }
  }
  if (warp == 0 && rank == 0 && chunk == g.chunks - 1 && on) put_two_floats(g.h_last + batch * g.dim + ch, state);
  if (lane == 0) sm100::bulk_wait_read_all();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    recurrence_backward_tma_kernel(const RecurrenceArgs g, const __grid_constant__ SequenceMaps maps) {
  constexpr int kRun = kRunBwd, kTile = kTileBwd, kStages = kStagesBwd<T>, kPart = kRun * kChan;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ Exchange ex;
  __shared__ float2 run_h[2][kWarps][32];
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % g.ranks, chunk = blockIdx.y;
  const int unit = blockIdx.x / g.ranks;
  const int batch = unit / g.channel_blocks, ch0 = unit % g.channel_blocks * kChan;
  const int64_t ch = ch0 + 2 * lane;
  const bool on = ch < g.dim, graded = g.grad != nullptr;
  const uint32_t bytes = (graded ? 3 : 2) * kPart * sizeof(T);
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t first = chunk * g.chunk_tiles, stop = min64(g.saved_tiles, first + g.chunk_tiles);
  T *ring = reinterpret_cast<T *>(dynamic) + size_t(warp) * kStages * 3 * kPart;
  auto stage = [&](int s) -> T * { return ring + s * 3 * kPart; };
  auto there = [&](int64_t k) { return k >= first && k * kTile + warp * kRun < g.steps; };
  auto fetch = [&](int64_t k, int s) {  // one lane
    if (!there(k)) return;
    const int t0 = static_cast<int>(k * kTile + warp * kRun);
    sm100::mbar_expect_tx(&full[warp][s], bytes);
    sm100::tma_load_3d(stage(s), &maps.gate, &full[warp][s], ch0, t0, batch);
    sm100::tma_load_3d(stage(s) + kPart, &maps.value, &full[warp][s], ch0, t0, batch);
    if (graded) sm100::tma_load_3d(stage(s) + 2 * kPart, &maps.grad, &full[warp][s], ch0, t0, batch);
  };
  auto flag_of = [&](int64_t k) -> uint32_t {
    const int64_t t = k * kTile + warp * kRun + lane;
    return reset != nullptr && k >= first && lane < kRun && t < g.steps ? __ldg(reset + t) : 0u;
  };
  auto before_of = [&](int64_t k) -> float2 {
    if (!there(k) || !on) return make_float2(0.f, 0.f);
    return two_floats(g.saved + (batch * g.saved_tiles + k) * g.dim + ch);
  };
  if (g.ranks > 1) cluster_arrive();
  if (threadIdx.x == 0) abort = 0;
  const int64_t k_first = stop - 1 - rank;
  // Stages are filled and used in order, one a tile that this warp has steps of: only the sequence's
  // last tile may be without.
  const bool skip = !there(k_first) && k_first >= first;
  const int64_t k_fill = skip ? k_first - g.ranks : k_first;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) sm100::mbar_init(&full[warp][s], 1);
    sm100::mbar_init_fence();
    sm100::fence_proxy_async_smem();
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(k_fill - int64_t(s) * g.ranks, s);
  }
  uint32_t flag = flag_of(k_first);
  float2 before = before_of(k_first);
  __syncthreads();

  float2 back = make_float2(0.f, 0.f);
  if (g.grad_last != nullptr && on) back = two_floats(g.grad_last + batch * g.dim + ch);
  if (chunk < g.chunks - 1) back = through_chunks<true, false>(g, batch, ch, on, on, chunk, back, ex);
  if (g.ranks > 1) cluster_wait();

  int buf = 0, s = 0, done = 0;
  uint32_t parity = 0;
  for (int64_t last = stop - 1, k = k_first; last >= first; last -= g.ranks, k -= g.ranks, buf ^= 1) {
    const bool here = there(k);
    const int n = here ? static_cast<int>(min64(kRun, g.steps - (k * kTile + warp * kRun))) : 0;
    const uint32_t cut = __ballot_sync(0xffffffffu, flag != 0);
    flag = flag_of(k - g.ranks);
    float2 h_in = before;
    before = before_of(k - g.ranks);
    const bool plain = n == kRun && cut == 0;
    if (here) sm100::mbar_wait(&full[warp][s], parity, &abort, &g_recurrence_error);
    T *rows = stage(s);
    float2 a[kRun], c[kRun], x[kRun], gt[kRun], p, h, r;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      gates2(unpack<T>(stage_raw<T>(rows + j * kChan, lane)), a[j], c[j]);
      x[j] = unpack<T>(stage_raw<T>(rows + kPart + j * kChan, lane));
      gt[j] = graded ? unpack<T>(stage_raw<T>(rows + 2 * kPart + j * kChan, lane)) : make_float2(0.f, 0.f);
    }
    scan_run_back<kRun>(a, c, x, gt, n, cut, plain, p, h, r);
    run_h[buf][warp][lane] = h;
    const float2 r_in = exchange<-1>(ex, buf, p, r, back, g.ranks, rank, reset != nullptr);
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w) {
      if (w < warp) h_in = apply_run(ex.p[buf][w][lane], h_in, run_h[buf][w][lane], reset != nullptr);
    }
    emit_run_back<kRun>(a, c, x, gt, n, cut, plain, h_in, r_in, [&](int j, float2 gf, float2 gx) {
      store_pair<T, true>(rows + j * kChan + 2 * lane, gf, true, true);
      store_pair<T, true>(rows + kPart + j * kChan + 2 * lane, gx, true, true);
    });
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (here) {
      if (lane == 0) {
        const int t0 = static_cast<int>(k * kTile + warp * kRun);
        tma_store_3d(&maps.out_gate, rows, ch0, t0, batch);
        tma_store_3d(&maps.out_value, rows + kPart, ch0, t0, batch);
        sm100::bulk_commit();
        // The stage before this one has been read by its stores: its next tile comes in.
        bulk_wait_read<1>();
        if (done > 0) fetch(k - int64_t(kStages - 1) * g.ranks, s == 0 ? kStages - 1 : s - 1);
      }
      ++done;
      if (++s == kStages) {
        s = 0;
        parity ^= 1;
      }
    }
  }
  if (warp == 0 && rank == 0 && chunk == 0 && g.grad_h0 != nullptr && on)
    put_two_floats(g.grad_h0 + batch * g.dim + ch, back);
  if (lane == 0) sm100::bulk_wait_read_all();
}

// The map of each chunk: (P, H) forward, (P, R) for the backward. Each warp scans an equal stretch of
// the chunk, the stretches are composed at the end.
template <typename T, bool PAIRED, bool FORWARD>
__global__ void __launch_bounds__(kThreads, 3) recurrence_map_kernel(const RecurrenceArgs g, int64_t chunk_steps) {
  constexpr int kRun = 8;
  __shared__ float2 run_p[kWarps][32], run_h[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = FORWARD ? blockIdx.y : blockIdx.y + 1;  // the last (first) chunk's map is not asked for
  const int64_t batch = blockIdx.x / g.channel_blocks;
  const Lane<PAIRED> at(blockIdx.x % g.channel_blocks, g.dim);
  const int64_t ch = at.ch;
  const bool on0 = at.on0, on1 = at.on1;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
  const T *other = FORWARD ? static_cast<const T *>(g.value) + batch * g.value_batch + at.from
                           : (g.grad != nullptr ? static_cast<const T *>(g.grad) + batch * g.steps * g.dim + at.from : nullptr);
  const int64_t other_step = FORWARD ? g.value_step : g.dim;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t share = chunk_steps / kWarps;  // a whole number of runs
  const int64_t begin = chunk * chunk_steps + warp * share, stop = min64(g.steps, begin + share);
  const float2 zero = make_float2(0.f, 0.f);
  float2 h = zero, p = make_float2(1.f, 1.f);
  const int64_t runs = begin < stop ? (stop - begin + kRun - 1) / kRun : 0;
  for (int64_t i = 0; i < runs; ++i) {
    const int64_t t0 = begin + (FORWARD ? i : runs - 1 - i) * kRun;
    const int n = static_cast<int>(min64(kRun, stop - t0));
    Raw<T> rf[kRun], ro[kRun] = {};
    const T *pf = gate + t0 * g.gate_step, *po = other + t0 * other_step;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      rf[j] = load_raw<T, PAIRED>(pf, at.second);
      if (other != nullptr) ro[j] = load_raw<T, PAIRED>(po, at.second);
      if (j + 1 < n) {  // steps past the end load the last one again
        pf += g.gate_step;
        po += other_step;
      }
    }
    const uint32_t cut = reset_bits(reset, t0, n);
#pragma unroll
    for (int i_j = 0; i_j < kRun; ++i_j) {
      const int j = FORWARD ? i_j : kRun - 1 - i_j;
      if (j < n) {
        const float2 f = unpack<T>(rf[j]), o = unpack<T>(ro[j]);
        float2 a, c;
        gates2(f, a, c);
        const bool here = (cut >> j) & 1u;
        if (FORWARD) {
          if (here) h = p = zero;
          h = fma2(a, h, mul2(c, o));
          p = mul2(p, a);
        } else {
          h = mul2(a, add2(o, h));
          p = mul2(p, a);
          if (here) h = p = zero;
        }
      }
    }
  }
  run_p[warp][lane] = p;
  run_h[warp][lane] = h;
  __syncthreads();
  if (warp == 0) {
    p = make_float2(1.f, 1.f);
    h = zero;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int w = FORWARD ? i : kWarps - 1 - i;
      h = apply_run(run_p[w][lane], h, run_h[w][lane], true);
      p = mul2(p, run_p[w][lane]);
    }
    float2 *m = g.maps + (batch * g.chunks + chunk) * g.dim + ch;
    if (on0) m[0] = make_float2(p.x, h.x);
    if (on1) m[kSecond<PAIRED>] = make_float2(p.y, h.y);
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
  float2 a, c;
  gates2(make_float2(to_f32<T>(gate[row * gate_row + ch]), 0.f), a, c);
  const float now = fmaf(a.x, before, c.x * to_f32<T>(value[row * value_row + ch]));
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

// How the tiles are shared out. While CTAs are idle: more of them a cluster, as far as there are tiles.
// With less than half the SMs busy even so and at least 4 tiles a chunk, chunks instead.
struct Plan {
  int ranks = 1, chunks = 1;
  int64_t chunk_tiles = 0;
};
Plan plan_for(int64_t units, int64_t tiles) {
  Plan p;
  p.chunk_tiles = tiles;
  while (p.ranks < kMaxCluster && units * p.ranks * 2 <= kSlots && p.ranks * 2 <= tiles) p.ranks *= 2;
  if (p.ranks == kMaxCluster && units * p.ranks <= kSlots / 4) {
    const int64_t each = std::max<int64_t>(4, ceil_div(tiles * units, kSlots));
    if (ceil_div(tiles, each) >= 2 * p.ranks) {
      p.ranks = 1;
      p.chunk_tiles = each;
      p.chunks = static_cast<int>(ceil_div(tiles, each));
    }
  }
  return p;
}
int64_t units_of(int64_t batch, int64_t dim) { return batch * ceil_div(dim, kChan); }
int64_t forward_tile(int dtype) { return kWarps * (dtype == TROPNN_B200_F32 ? kRunFwd<float> : kRunFwd<__half>); }

// A [batch, steps, dim] tensor (strides in elements) in boxes of `run` steps x 64 channels. False where
// TMA cannot take it.
bool sequence_map(CUtensorMap *map, const void *ptr, int dtype, int64_t batch, int64_t steps, int64_t dim,
                  int64_t batch_stride, int64_t step_stride, int run) {
  const int64_t size = dtype == TROPNN_B200_F32 ? 4 : 2;
  // The stride of a dimension of one element is never used, but has to be a valid one.
  if (steps == 1) step_stride = ceil_div(dim, 16) * 16;
  if (batch == 1) batch_stride = steps * step_stride;
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0 || dim > 0x7fffffffLL || steps > 0x7fffffffLL || batch > 0x7fffffffLL) return false;
  for (int64_t stride : {step_stride, batch_stride})
    if (stride <= 0 || stride * size % 16 != 0 || stride * size >= (1LL << 40)) return false;
  sm100::EncodeTiledFn fn = nullptr;
  if (sm100::encode_fn(&fn) != TROPNN_B200_OK) return false;
  const CUtensorMapDataType type = dtype == TROPNN_B200_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == TROPNN_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(steps), static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(step_stride * size), static_cast<cuuint64_t>(batch_stride * size)};
  const cuuint32_t box[3] = {kChan, static_cast<cuuint32_t>(run), 1};
  const cuuint32_t each[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void *>(ptr), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FORWARD, typename T, bool PAIRED>
int launch_typed(const char *what, RecurrenceArgs g, int dtype, int64_t batch, const Plan &plan, cudaStream_t stream) {
  const unsigned units = static_cast<unsigned>(batch * g.channel_blocks);
  if (plan.chunks > 1) {
    constexpr int64_t tile = FORWARD ? kWarps * kRunFwd<T> : kTileBwd;
    recurrence_map_kernel<T, PAIRED, FORWARD>
        <<<dim3(units, static_cast<unsigned>(plan.chunks - 1)), kThreads, 0, stream>>>(g, plan.chunk_tiles * tile);
    TB_CHECK(check_launch(what));
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(units * static_cast<unsigned>(plan.ranks), static_cast<unsigned>(plan.chunks));
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(plan.ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  if constexpr (PAIRED) {
    SequenceMaps maps{};
    constexpr int run = FORWARD ? kRunFwd<T> : kRunBwd;
    const int64_t steps = g.steps, dim = g.dim;
    bool fits = steps > 0 && sequence_map(&maps.gate, g.gate, dtype, batch, steps, dim, g.gate_batch, g.gate_step, run) &&
                sequence_map(&maps.value, g.value, dtype, batch, steps, dim, g.value_batch, g.value_step, run);
    if (FORWARD) {
      fits = fits && sequence_map(&maps.out_value, g.h, dtype, batch, steps, dim, steps * dim, dim, run);
    } else {
      fits = fits && (g.grad == nullptr || sequence_map(&maps.grad, g.grad, dtype, batch, steps, dim, steps * dim, dim, run)) &&
             sequence_map(&maps.out_gate, g.grad_gate, dtype, batch, steps, dim, steps * dim, dim, run) &&
             sequence_map(&maps.out_value, g.grad_value, dtype, batch, steps, dim, steps * dim, dim, run);
    }
    if (fits) {
      config.dynamicSmemBytes = kRingBytes<T, FORWARD>;
      const void *kernel = FORWARD ? reinterpret_cast<const void *>(recurrence_forward_tma_kernel<T>)
                                   : reinterpret_cast<const void *>(recurrence_backward_tma_kernel<T>);
      // The static part counts too: above 48 KB in all the kernel has to be told.
      TB_CHECK(ensure_dynamic_smem(kernel, std::max<size_t>(config.dynamicSmemBytes, 49 * 1024), what));
      void *args[] = {&g, &maps};
      cudaLaunchKernelExC(&config, kernel, args);
      return check_launch(what);
    }
  }
  if (FORWARD) cudaLaunchKernelEx(&config, recurrence_forward_kernel<T, PAIRED>, static_cast<const RecurrenceArgs>(g));
  else cudaLaunchKernelEx(&config, recurrence_backward_kernel<T, PAIRED>, static_cast<const RecurrenceArgs>(g));
  return check_launch(what);
}

template <bool FORWARD>
int launch_recurrence(const char *what, RecurrenceArgs g, int dtype, int64_t batch, bool pair, void *workspace,
                      size_t workspace_bytes, cudaStream_t stream) {
  const int64_t tile = FORWARD ? forward_tile(dtype) : kTileBwd;
  const Plan plan = plan_for(batch * g.channel_blocks, ceil_div(g.steps, tile));
  const size_t need = plan.chunks > 1 ? static_cast<size_t>(batch * plan.chunks * g.dim) * sizeof(float2) : 0;
  TB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), TROPNN_B200_ERR_WORKSPACE,
             "%s: %zu bytes of workspace, %zu needed", what, workspace_bytes, need);
  g.ranks = plan.ranks;
  g.chunks = plan.chunks;
  g.chunk_tiles = plan.chunk_tiles;
  g.maps = static_cast<float2 *>(workspace);
  if (dtype == TROPNN_B200_F32)
    return pair ? launch_typed<FORWARD, float, true>(what, g, dtype, batch, plan, stream)
                : launch_typed<FORWARD, float, false>(what, g, dtype, batch, plan, stream);
  if (dtype == TROPNN_B200_F16)
    return pair ? launch_typed<FORWARD, __half, true>(what, g, dtype, batch, plan, stream)
                : launch_typed<FORWARD, __half, false>(what, g, dtype, batch, plan, stream);
  return pair ? launch_typed<FORWARD, __nv_bfloat16, true>(what, g, dtype, batch, plan, stream)
              : launch_typed<FORWARD, __nv_bfloat16, false>(what, g, dtype, batch, plan, stream);
}

}  // namespace

// Reads and clears this file's device error word (a wait for a tile that ran out).
int read_recurrence_error(int *value) {
  int v = 0;
  cudaError_t err = cudaMemcpyFromSymbol(&v, g_recurrence_error, sizeof(int));
  if (err != cudaSuccess) return set_error(TROPNN_B200_ERR_LAUNCH, "reading the device error word: %s", cudaGetErrorString(err));
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_recurrence_error, &zero, sizeof(int));
  }
  *value = v;
  return TROPNN_B200_OK;
}

}  // namespace tropnn_b200

using namespace tropnn_b200;

extern "C" {

size_t tropnn_b200_recurrence_saved_size(int64_t batch, int64_t steps, int64_t dim) {
  if (batch <= 0 || steps <= 0 || dim <= 0) return 0;
  return static_cast<size_t>(batch * ceil_div(steps, kTileBwd) * dim) * sizeof(float);
}

size_t tropnn_b200_recurrence_workspace_size(int64_t batch, int64_t steps, int64_t dim, int dtype) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || !is_float_dtype(dtype)) return 0;
  const int64_t units = units_of(batch, dim);
  const Plan f = plan_for(units, ceil_div(steps, forward_tile(dtype))), b = plan_for(units, ceil_div(steps, kTileBwd));
  const int chunks = std::max(f.chunks, b.chunks);
  return chunks > 1 ? static_cast<size_t>(batch * chunks * dim) * sizeof(float2) : 0;
}

int tropnn_b200_recurrence_forward(const void *gate, int64_t gate_batch_stride, int64_t gate_step_stride,
                                   const void *value, int64_t value_batch_stride, int64_t value_step_stride, int dtype,
                                   const float *h0, const uint8_t *reset, int64_t batch, int64_t steps, int64_t dim,
                                   void *h, float *h_last, float *saved, size_t saved_bytes, void *workspace,
                                   size_t workspace_bytes, void *stream) {
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
  TB_CHECK((launch_recurrence<true>(what, g, dtype, batch, pair, workspace, workspace_bytes, as_stream(stream))));
  return clear_error();
}

int tropnn_b200_recurrence_backward(const void *gate, int64_t gate_batch_stride, int64_t gate_step_stride,
                                    const void *value, int64_t value_batch_stride, int64_t value_step_stride, int dtype,
                                    const uint8_t *reset, int64_t batch, int64_t steps, int64_t dim, const float *saved,
                                    size_t saved_bytes, const void *grad, const float *grad_last, void *grad_gate,
                                    void *grad_value, float *grad_h0, void *workspace, size_t workspace_bytes,
                                    void *stream) {
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
  TB_CHECK((launch_recurrence<false>(what, g, dtype, batch, pair, workspace, workspace_bytes, as_stream(stream))));
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
