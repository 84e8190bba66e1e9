// Gated linear recurrence over token sequences: forward, backward and the single-token step.
//
//   a_t = sigmoid(f_t), c_t = 1 - a_t = sigmoid(-f_t)          (per channel)
//   h_t = keep_t a_t h_{t-1} + c_t x_t                          (keep_t = 0 at a reset, else 1)
//
// The recurrence is linear, so a stretch of steps maps the state before it to P h + H with P the
// product of its gates (marked where a reset cuts it). A lane has two neighbouring channels, a warp 64; both are computed in f32x2
// instructions. Two schemes, each bound by issue slots and latencies before HBM:
//  - tiles (the forward where the channels fill the GPU: 28 blocks of 64 and more, in f32 19, rows of the
//    batch counted; and of short sequences): a warp scans a run of steps in registers, the runs' maps are exchanged, and the run is scanned again from the state
//    before it. Gate and value are read and turned into gates once; every tile waits for a barrier.
//  - segments (the backward, and the forward of few channels): each warp has a stretch of the sequence
//    of its own and goes over it twice without waiting for any other, first for the stretch's map, then,
//    with the state before it composed, for the results. The second pass finds its inputs in L2 as far
//    as they fit (126 MB). The one exchange goes through the shared memory of a cluster of up to 8 CTAs,
//    or through global memory between two launches.
// Measured at 8 x 2048 x 1024 bf16: forward 29 us by tiles (3.5 TB/s of reads and writes), 41 us by
// segments; backward 44 us by segments (3.8 TB/s), 58 us by tiles. At 1 x 65536 x 256 f16: forward 37 us
// and backward 45 us by segments in two launches, 169 and 231 us by tiles and segments of one cluster.
// At 3 x 1531 x 777 f32, whose rows allow neither pairs nor TMA: 19 and 43 us.
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed.cuh"
#include "sm100.cuh"

namespace tropnn_b200 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChan = 64;                    // channels of a CTA, two a lane
constexpr int kRun = 8;  // steps that a warp takes at once, and the distance of the saved states
constexpr int kMaxCluster = 8;
constexpr int kMapSlots = kWarps + 1;  // maps of a chunk in global memory: its segments', and its own

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

// a and c = 1 - a. The smaller one, m = e / (1 + e) with e = exp(-|f|), does not cancel: it is off by
// |f| 2^-24 of itself (the rounding of exp's argument) and some 2^-22 (the approximate units), and is 0
// where e is below 2^-126. The larger is 1 - m, the f32 next to it.
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

// P h + H. A stretch that a reset cuts takes nothing of h, whatever h or its own P is: it says so by P =
// kCut. A product of gates is never negative, but is 0 where it underflows (128 gates of an untrained
// layer often do), and then a NaN in h stays one. `cuts`: resets are given.
constexpr float kCut = -1.f;
__device__ __forceinline__ float2 apply_run(float2 p, float2 h, float2 add, bool cuts) {
  if (!cuts) return fma2(p, h, add);
  return make_float2(p.x < 0.f ? add.x : fmaf(p.x, h.x, add.x), p.y < 0.f ? add.y : fmaf(p.y, h.y, add.y));
}
// P of two stretches, one after the other.
__device__ __forceinline__ float2 join_runs(float2 p, float2 q, bool cuts) {
  if (!cuts) return mul2(p, q);
  return make_float2(p.x < 0.f || q.x < 0.f ? kCut : p.x * q.x, p.y < 0.f || q.y < 0.f ? kCut : p.y * q.y);
}

struct RecurrenceArgs {
  const void *gate, *value;
  int64_t gate_batch, gate_step, value_batch, value_step;
  const float *h0;
  const uint8_t *reset;
  int64_t steps, dim, runs;  // runs: ceil(steps / kRun)
  int channel_blocks;
  int chunks;            // of the sequence, a CTA each
  int64_t segment_runs;  // of a warp; a chunk is kWarps segments
  float2 *maps;          // two launches: (P, H) or (P, R) of [batch, chunk, kMapSlots, dim]
  void *h;
  float *h_last;
  float *saved;  // [batch, runs, dim]: the state before each run; NULL: not kept
  // backward
  const void *grad;
  const float *grad_last;
  void *grad_gate, *grad_value;
  float *grad_h0;
};

// What a launch does: both passes with a cluster's exchange between them (the backward), or one of the
// two.
enum Pass { kBoth = 0, kMaps = 1, kApply = 2 };

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Neighbours in an f32 array that may start anywhere.
__device__ __forceinline__ float2 two_floats(const float *p, int second) { return make_float2(__ldg(p), __ldg(p + second)); }

// Maps of the CTA's segments and of the cluster's chunks, two lane channels each.
struct Exchange {
  float2 p[kWarps][32], h[kWarps][32];
  float4 rank[kMaxCluster][32];
};

// Hands this warp's (p, h) around and returns the state before its segment, from the state before the
// sequence. FORWARD: segments follow one another by warp and chunk, else from the last back.
template <bool FORWARD, bool PAIRED, int PASS>
__device__ __forceinline__ float2 exchange(const RecurrenceArgs &g, int64_t batch, const Lane<PAIRED> &at, int chunk, float2 p,
                                           float2 h, float2 state, Exchange &ex) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool cuts = g.reset != nullptr;
  const int place = FORWARD ? chunk : g.chunks - 1 - chunk;  // chunks before this one
  const int order = FORWARD ? warp : kWarps - 1 - warp;      // segments of the chunk before this one
  if (PASS != kApply) {
    ex.p[order][lane] = p;
    ex.h[order][lane] = h;
    __syncthreads();
    if (PASS == kMaps ? order == kWarps - 1 : warp < g.chunks) {  // the chunk's map
      float2 cp = make_float2(1.f, 1.f), ch = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ch = apply_run(ex.p[w][lane], ch, ex.h[w][lane], cuts);
        cp = join_runs(cp, ex.p[w][lane], cuts);
      }
      if (PASS == kBoth) {
        if (g.chunks > 1)
          *cooperative_groups::this_cluster().map_shared_rank(&ex.rank[place][lane], warp) = make_float4(cp.x, cp.y, ch.x, ch.y);
      } else {
        float2 *m = g.maps + ((batch * g.chunks + chunk) * kMapSlots + kWarps) * g.dim + at.ch;
        if (at.on0) m[0] = make_float2(cp.x, ch.x);
        if (at.on1) m[kSecond<PAIRED>] = make_float2(cp.y, ch.y);
      }
    }
    if (PASS == kMaps) {
      float2 *m = g.maps + ((batch * g.chunks + chunk) * kMapSlots + order) * g.dim + at.ch;
      if (at.on0) m[0] = make_float2(p.x, h.x);
      if (at.on1) m[kSecond<PAIRED>] = make_float2(p.y, h.y);
      return state;
    }
    if (g.chunks > 1) {
      cluster_arrive();
      cluster_wait();
      for (int r = 0; r < place; ++r) {
        const float4 m = ex.rank[r][lane];
        state = apply_run(make_float2(m.x, m.y), state, make_float2(m.z, m.w), cuts);
      }
    }
    for (int w = 0; w < order; ++w) state = apply_run(ex.p[w][lane], state, ex.h[w][lane], cuts);
    return state;
  }
  // From global memory: the chunks before this one, a share a warp, then this one's segments.
  auto map_at = [&](int c, int slot, float2 &mp, float2 &mh) {
    const float2 *m = g.maps + ((batch * g.chunks + (FORWARD ? c : g.chunks - 1 - c)) * kMapSlots + slot) * g.dim + at.from;
    const float2 a = __ldg(m), b = __ldg(m + at.second);
    mp = make_float2(a.x, b.x);
    mh = make_float2(a.y, b.y);
  };
  const int share = (place + kWarps - 1) / kWarps, first = min(warp * share, place), stop = min(first + share, place);
  p = make_float2(1.f, 1.f);
  h = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int c = first; c < stop; ++c) {
    float2 mp, mh;
    map_at(c, kWarps, mp, mh);
    h = apply_run(mp, h, mh, cuts);
    p = join_runs(mp, p, cuts);
  }
  ex.p[warp][lane] = p;
  ex.h[warp][lane] = h;
  float2 own_p[kWarps - 1], own_h[kWarps - 1];
#pragma unroll
  for (int w = 0; w < kWarps - 1; ++w)
    if (w < order) map_at(place, w, own_p[w], own_h[w]);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) state = apply_run(ex.p[w][lane], state, ex.h[w][lane], cuts);
#pragma unroll
  for (int w = 0; w < kWarps - 1; ++w)
    if (w < order) state = apply_run(own_p[w], state, own_h[w], cuts);
  return state;
}

// The reset flags of a run as bits, from the byte that each lane loaded ahead.
__device__ __forceinline__ uint32_t flag_of(const uint8_t *reset, int t0, int steps) {
  const int t = t0 + static_cast<int>(threadIdx.x & 31);
  return reset != nullptr && (threadIdx.x & 31) < kRun && t < steps ? __ldg(reset + t) : 0u;
}

// Tensor maps of the TMA form.
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
__device__ __forceinline__ float2 stage_pair(const T *row, int lane) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    const float2 q = reinterpret_cast<const float2 *>(row)[lane];
    r.a = q.x;
    r.b = q.y;
  } else {
    r.v = reinterpret_cast<const uint32_t *>(row)[lane];
  }
  return unpack<T>(r);
}

// How a warp's runs of up to three tensors come in and its results go out. TMA: a ring of stages in
// shared memory a warp, filled two or three runs ahead across both passes; results are written over a
// stage's inputs and stored from there, rows and channels that are not there come as zeros and are not
// written. Needs rows 16 bytes aligned (dim and strides multiples of 8 16-bit or 4 f32 elements). Else
// plain loads, a run ahead in registers, by pairs of channels where alignment allows.
template <typename T, int TENSORS>
constexpr int kStages = TENSORS == 3 && sizeof(T) == 4 ? 2 : 3;
template <typename T, int TENSORS>
constexpr size_t kRingBytes = size_t(kWarps) * kStages<T, TENSORS> * TENSORS * kRun * kChan * sizeof(T);

template <typename T, int TENSORS, bool TMA, bool PAIRED>
struct Stream {
  static constexpr int kDeep = kStages<T, TENSORS>;
  // TMA
  T *ring;
  uint64_t *full;
  int *abort;
  const CUtensorMap *maps[TENSORS];
  int ch0, batch, s = 0;
  uint32_t parity = 0;
  bool stored = false, alive = true;
  // plain
  const T *from[TENSORS];
  int64_t stride[TENSORS];
  int steps, second;
  Raw<T> raw[TMA ? 1 : TENSORS][TMA ? 1 : kRun];

  __device__ __forceinline__ T *rows(int tensor) { return ring + (s * TENSORS + tensor) * kRun * kChan; }
  // Starts the loads of the tensors in `which` (a bit each) of the run at t0, `ahead` stages on.
  __device__ __forceinline__ void fetch(int t0, uint32_t which, int ahead) {
    if constexpr (TMA) {
      if ((threadIdx.x & 31) == 0 && alive) {
        int at = s + ahead;
        if (at >= kDeep) at -= kDeep;
        sm100::mbar_expect_tx(&full[at], __popc(which) * kRun * kChan * sizeof(T));
#pragma unroll
        for (int i = 0; i < TENSORS; ++i)
          if ((which >> i) & 1u)
            sm100::tma_load_3d(ring + (at * TENSORS + i) * kRun * kChan, maps[i], &full[at], ch0, t0, batch);
      }
    } else {
      // Steps past the end load the last one again.
      const int most = steps - 1 - t0;
#pragma unroll
      for (int i = 0; i < TENSORS; ++i) {
        if (!((which >> i) & 1u)) continue;
        const T *p = from[i] + t0 * stride[i];
        if (most >= kRun - 1) {
#pragma unroll
          for (int j = 0; j < kRun; ++j, p += stride[i]) raw[i][j] = load_raw<T, PAIRED>(p, second);
        } else {
#pragma unroll
          for (int j = 0; j < kRun; ++j) raw[i][j] = load_raw<T, PAIRED>(p + min(j, most) * stride[i], second);
        }
      }
    }
  }
  // The stage of the run with `left` runs (it included) to come has arrived. Where a wait runs out, a lane
  // waits no more, and lane 0, which issues the copies, sees those on their way out and starts no others;
  // the warp goes on with what lies in its ring, so that it meets the block at every barrier.
  __device__ __forceinline__ void wait(int left) {
    if constexpr (TMA) {
      if (!alive || sm100::mbar_wait(&full[s], parity, abort, &g_recurrence_error)) return;
      alive = false;
      if ((threadIdx.x & 31) != 0) return;
      for (int n = min(kDeep - (stored ? 1 : 0), left), at = s, p = parity; n > 0; --n) {
        sm100::mbar_drain(&full[at], p);
        if (++at == kDeep) {
          at = 0;
          p ^= 1;
        }
      }
    }
  }
  __device__ __forceinline__ float2 get(int tensor, int j) {
    if constexpr (TMA) return stage_pair<T>(rows(tensor) + j * kChan, threadIdx.x & 31);
    else return unpack<T>(raw[tensor][j]);
  }
  // The stage has been read.
  __device__ __forceinline__ void next() {
    if constexpr (TMA) {
      if (++s == kDeep) {
        s = 0;
        parity ^= 1;
      }
    }
  }
};

// Items of a warp: its segment's runs for the maps, then again for the results, in one order. Steps are
// below 2^31.
template <bool FORWARD, int PASS>
struct Items {
  int first, count, total;  // runs, items
  __device__ __forceinline__ Items(const RecurrenceArgs &g, int chunk, int warp) {
    const int64_t runs = g.runs, at = min64((int64_t(chunk) * kWarps + warp) * g.segment_runs, runs);
    first = static_cast<int>(at);
    count = static_cast<int>(min64(g.segment_runs, runs - at));
    total = PASS == kBoth ? 2 * count : count;
  }
  __device__ __forceinline__ int start(int i) const {  // first step of item i
    const int n = PASS == kBoth && i >= count ? i - count : i;
    return (FORWARD ? first + n : first + count - 1 - n) * kRun;
  }
};

template <typename T, bool TMA, bool PAIRED, int PASS>
__global__ void __launch_bounds__(kThreads, TMA && sizeof(T) == 2 ? 3 : 2)
    recurrence_forward_kernel(const RecurrenceArgs g, const __grid_constant__ SequenceMaps maps) {
  static_assert(PASS != kBoth, "a forward in one launch goes by tiles");
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ Exchange ex;
  __shared__ uint64_t full[kWarps][4];
  __shared__ int abort;
  using In = Stream<T, 2, TMA, PAIRED>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.x / g.chunks, chunk = blockIdx.x - unit * g.chunks;
  const int64_t batch = unit / g.channel_blocks;
  const int block = unit - static_cast<int>(batch) * g.channel_blocks;
  const Lane<PAIRED> at(block, g.dim);
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const Items<true, PASS> items(g, chunk, warp);
  const int total = items.total, steps = static_cast<int>(g.steps);

  In in;
  if constexpr (TMA) {
    in.ring = reinterpret_cast<T *>(dynamic) + size_t(warp) * In::kDeep * 2 * kRun * kChan;
    in.full = full[warp];
    in.abort = &abort;
    in.maps[0] = &maps.gate;
    in.maps[1] = &maps.value;
    in.ch0 = block * kChan;
    in.batch = static_cast<int>(batch);
    if (threadIdx.x == 0) abort = 0;
    if (lane == 0) {
#pragma unroll
      for (int s = 0; s < In::kDeep; ++s) sm100::mbar_init(&full[warp][s], 1);
      sm100::mbar_init_fence();
      sm100::fence_proxy_async_smem();
    }
    __syncthreads();
  } else {
    in.from[0] = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
    in.from[1] = static_cast<const T *>(g.value) + batch * g.value_batch + at.from;
    in.stride[0] = g.gate_step;
    in.stride[1] = g.value_step;
    in.steps = steps;
    in.second = at.second;
  }
  const int ahead = TMA ? In::kDeep : 1;
  for (int i = 0; i < ahead; ++i)
    if (i < total) in.fetch(items.start(i), 3, i);
  uint32_t flag = total > 0 ? flag_of(reset, items.start(0), steps) : 0;

  float2 h = make_float2(0.f, 0.f), p = make_float2(1.f, 1.f);
  uint32_t was_cut = 0;
  int item = 0;
  // One run: step(j, a, c x) for each of its steps, then the loads of a later one.
  auto gates_of = [&](float2 (&a)[kRun], float2 (&b)[kRun]) {
    in.wait(total - item);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      float2 c;
      gates2(in.get(0, j), a[j], c);
      b[j] = mul2(c, in.get(1, j));
    }
  };
  auto flags = [&]() -> uint32_t {
    if (reset == nullptr) return 0;
    const uint32_t cut = __ballot_sync(0xffffffffu, flag != 0);
    flag = item + 1 < total ? flag_of(reset, items.start(item + 1), steps) : 0;
    return cut;
  };
  if (PASS != kApply) {
    for (; item < items.count; ++item) {
      const int t0 = items.start(item);
      const int n = min(kRun, steps - t0);
      const uint32_t cut = flags();
      float2 a[kRun], b[kRun];
      gates_of(a, b);
      if constexpr (TMA) __syncwarp();  // all lanes have read the stage
      if (item + ahead < total) in.fetch(items.start(item + ahead), 3, 0);
      in.next();
      if (n == kRun && cut == 0) {
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          h = fma2(a[j], h, b[j]);
          p = mul2(p, a[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          if (j < n) {
            if ((cut >> j) & 1u) h = make_float2(0.f, 0.f);
            h = fma2(a[j], h, b[j]);
            p = mul2(p, a[j]);
          }
        }
        was_cut |= cut;
      }
    }
    if (was_cut != 0) p = both(kCut);
  }
  float2 state = make_float2(0.f, 0.f);
  if (g.h0 != nullptr) state = two_floats(g.h0 + batch * g.dim + at.from, at.second);
  state = exchange<true, PAIRED, PASS>(g, batch, at, chunk, p, h, state, ex);
  if (PASS == kMaps) return;

  T *out = static_cast<T *>(g.h) + batch * g.steps * g.dim + at.ch;
  for (; item < total; ++item) {
    const int t0 = items.start(item);
    const int n = min(kRun, steps - t0);
    const uint32_t cut = flags();
    float2 a[kRun], b[kRun];
    gates_of(a, b);
    if constexpr (!TMA)
      if (item + 1 < total) in.fetch(items.start(item + 1), 3, 0);
    if (g.saved != nullptr) {
      float *s = g.saved + (batch * g.runs + t0 / kRun) * g.dim + at.ch;
      if (at.on0) s[0] = state.x;
      if (at.on1) s[kSecond<PAIRED>] = state.y;
    }
    auto put = [&](int j) {
      if constexpr (TMA) store_pair<T, true>(in.rows(1) + j * kChan + 2 * lane, state, true, true);
      else store_pair<T, PAIRED>(out + int64_t(t0 + j) * g.dim, state, at.on0, at.on1);
    };
    if (n == kRun && cut == 0) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        state = fma2(a[j], state, b[j]);
        put(j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (j < n) {
          if ((cut >> j) & 1u) state = make_float2(0.f, 0.f);
          state = fma2(a[j], state, b[j]);
          put(j);
        }
      }
    }
    if constexpr (TMA) {
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (in.alive) tma_store_3d(&maps.out_value, in.rows(1), in.ch0, t0, in.batch);
        sm100::bulk_commit();
        bulk_wait_read<1>();  // the stage before this one has been read by its store
      }
      // That stage's next run comes in; the first run's stage has no store before it.
      if (in.stored && item - 1 + In::kDeep < total) in.fetch(items.start(item - 1 + In::kDeep), 3, In::kDeep - 1);
      in.stored = true;
    }
    in.next();
  }
  if (warp == kWarps - 1 && chunk == g.chunks - 1) {
    float *last = g.h_last + batch * g.dim + at.ch;
    if (at.on0) last[0] = state.x;
    if (at.on1) last[kSecond<PAIRED>] = state.y;
  }
  if (TMA && lane == 0) sm100::bulk_wait_read_all();
}

// Forward with channels enough to fill the GPU: tiles in the order of the sequence. A CTA's 8 warps take a
// tile of 8 runs of a warp each, scan them in registers for their maps, exchange those and scan again
// from the state before each run: gate and value are read and turned into gates once, at the price of a
// barrier a tile. A cluster of up to 8 CTAs takes as many consecutive tiles at once and exchanges their
// maps through distributed shared memory; the next tiles' loads are under way meanwhile.
// Steps of a warp's run: what leaves room for the next tile's values in 128 registers a thread.
template <typename T>
constexpr int kTileRun = sizeof(T) == 2 ? 16 : 8;
constexpr int kTileStages = 3;
template <typename T>
constexpr size_t kTileRingBytes = size_t(kWarps) * kTileStages * 2 * kTileRun<T> * kChan * sizeof(T);

__device__ __forceinline__ void put_two_floats(float *p, float2 v) {
  p[0] = v.x;
  p[1] = v.y;
}

// Exchange of a tile: (P, H) of the CTA's warps and of the cluster's CTAs, two lane channels each.
struct TileExchange {
  float2 p[2][kWarps][32], h[2][kWarps][32];
  float4 rank[2][kMaxCluster][32];
};

// Hands this warp's (p, h) around: returns the state before its run, and moves `state` past the cluster's
// tiles.
__device__ __forceinline__ float2 tile_exchange(TileExchange &ex, int buf, float2 p, float2 h, float2 &state, int ranks, int rank,
                                           bool cuts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ex.p[buf][warp][lane] = p;
  ex.h[buf][warp][lane] = h;
  __syncthreads();
  float2 in = state;
  if (ranks == 1) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) in = state;
      state = apply_run(ex.p[buf][w][lane], state, ex.h[buf][w][lane], cuts);
    }
    return in;
  }
  if (warp < ranks) {  // the CTA's map, to one CTA a warp
    float2 cp = make_float2(1.f, 1.f), ch = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 pw = ex.p[buf][w][lane];
      ch = apply_run(pw, ch, ex.h[buf][w][lane], cuts);
      cp = join_runs(cp, pw, cuts);
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
  for (int w = 0; w < kWarps - 1; ++w) {
    if (w < warp) in = apply_run(ex.p[buf][w][lane], in, ex.h[buf][w][lane], cuts);
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
        if ((cut >> j) & 1u) h = zero;
        h = fma2(a[j], h, b[j]);
        p = mul2(p, a[j]);
      }
    }
    if (cut != 0) p = both(kCut);
  }
}
// The run from the state before it: save(j, h_{j-1}) at every kRun-th step, store(j, h_j).
template <int RUN, typename Save, typename Store>
__device__ __forceinline__ void emit_run(const float2 (&a)[RUN], const float2 (&b)[RUN], int n, uint32_t cut, bool plain,
                                         float2 in, Save save, Store store) {
  if (plain) {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j % kRun == 0) save(j, in);
      in = fma2(a[j], in, b[j]);
      store(j, in);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
      if (j < n) {
        if (j % kRun == 0) save(j, in);
        if ((cut >> j) & 1u) in = make_float2(0.f, 0.f);
        in = fma2(a[j], in, b[j]);
        store(j, in);
      }
    }
  }
}
template <typename T, bool PAIRED>
__global__ void __launch_bounds__(kThreads, 2) recurrence_tiles_kernel(const RecurrenceArgs g) {
  constexpr int kLong = kTileRun<T>, kTile = kWarps * kLong;
  __shared__ TileExchange ex;
  const int warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % g.chunks;
  const int unit = blockIdx.x / g.chunks;
  const int64_t batch = unit / g.channel_blocks;
  const Lane<PAIRED> at(unit % g.channel_blocks, g.dim);
  const int64_t ch = at.ch;
  const bool on0 = at.on0, on1 = at.on1;
  const T *gate = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
  const T *value = static_cast<const T *>(g.value) + batch * g.value_batch + at.from;
  T *out = static_cast<T *>(g.h) + batch * g.steps * g.dim + ch;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t stop = g.steps;
  if (g.chunks > 1) cluster_arrive();

  Raw<T> rf[kLong], rx[kLong];
  auto load = [&](int64_t t0) {
    if (t0 >= stop) return;
    // Steps past the end load the last one again.
    const int64_t most = stop - 1 - t0;
    const T *pf = gate + t0 * g.gate_step, *px = value + t0 * g.value_step;
    if (most >= kLong - 1) {
#pragma unroll
      for (int j = 0; j < kLong; ++j, pf += g.gate_step, px += g.value_step) {
        rf[j] = load_raw<T, PAIRED>(pf, at.second);
        rx[j] = load_raw<T, PAIRED>(px, at.second);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kLong; ++j) {
        rf[j] = load_raw<T, PAIRED>(pf + min64(j, most) * g.gate_step, at.second);
        rx[j] = load_raw<T, PAIRED>(px + min64(j, most) * g.value_step, at.second);
      }
    }
  };
  load(rank * kTile + warp * kLong);
  float2 state = make_float2(0.f, 0.f);  // the state before the cluster's tiles, the same in every warp
  if (g.h0 != nullptr) {
    const float *p = g.h0 + batch * g.dim + ch;
    if (on0) state.x = p[0];
    if (on1) state.y = p[kSecond<PAIRED>];
  }
  if (g.chunks > 1) cluster_wait();

  int buf = 0;
  for (int64_t tile = 0; tile < stop; tile += int64_t(g.chunks) * kTile, buf ^= 1) {
    const int64_t t0 = tile + rank * kTile + warp * kLong;
    const int n = static_cast<int>(t0 >= stop ? 0 : min64(kLong, stop - t0));
    const uint32_t cut = reset_bits(reset, t0, n);
    const bool plain = n == kLong && cut == 0;
    float2 a[kLong], b[kLong], p, h;
#pragma unroll
    for (int j = 0; j < kLong; ++j) {
      float2 c;
      gates2(unpack<T>(rf[j]), a[j], c);
      b[j] = mul2(c, unpack<T>(rx[j]));
    }
    scan_run<kLong>(a, b, n, cut, plain, p, h);
    load(t0 + int64_t(g.chunks) * kTile);
    const float2 in = tile_exchange(ex, buf, p, h, state, g.chunks, rank, reset != nullptr);
    T *po = out + t0 * g.dim;
    auto save = [&](int j, float2 v) {
      if (g.saved == nullptr) return;
      float *s = g.saved + (batch * g.runs + (t0 + j) / kRun) * g.dim + ch;
      if (on0) s[0] = v.x;
      if (on1) s[kSecond<PAIRED>] = v.y;
    };
    emit_run<kLong>(a, b, n, cut, plain, in, save, [&](int, float2 v) {
      store_pair<T, PAIRED>(po, v, on0, on1);
      po += g.dim;
    });
  }
  if (warp == 0 && rank == 0) {
    float *p = g.h_last + batch * g.dim + ch;
    if (on0) p[0] = state.x;
    if (on1) p[kSecond<PAIRED>] = state.y;
  }
}

// The same with TMA: each warp has a ring of its own.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    recurrence_tiles_tma_kernel(const RecurrenceArgs g, const __grid_constant__ SequenceMaps maps) {
  constexpr int kLong = kTileRun<T>, kTile = kWarps * kLong, kStages = kTileStages;
  constexpr uint32_t kBytes = 2 * kLong * kChan * sizeof(T);
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ TileExchange ex;
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % g.chunks;
  const int unit = blockIdx.x / g.chunks;
  const int batch = unit / g.channel_blocks, ch0 = unit % g.channel_blocks * kChan;
  const int64_t ch = ch0 + 2 * lane;
  const bool on = ch < g.dim;
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const int64_t stop = g.steps;
  const int64_t stride = int64_t(g.chunks) * kTile;
  T *ring = reinterpret_cast<T *>(dynamic) + size_t(warp) * kStages * 2 * kLong * kChan;
  auto stage = [&](int s) -> T * { return ring + s * 2 * kLong * kChan; };
  auto fetch = [&](int64_t t0, int s) {  // one lane
    if (t0 >= stop) return;
    sm100::mbar_expect_tx(&full[warp][s], kBytes);
    sm100::tma_load_3d(stage(s), &maps.gate, &full[warp][s], ch0, static_cast<int>(t0), batch);
    sm100::tma_load_3d(stage(s) + kLong * kChan, &maps.value, &full[warp][s], ch0, static_cast<int>(t0), batch);
  };
  auto flag_of = [&](int64_t t0) -> uint32_t {
    return reset != nullptr && lane < kLong && t0 + lane < stop ? __ldg(reset + t0 + lane) : 0u;
  };
  if (g.chunks > 1) cluster_arrive();
  if (threadIdx.x == 0) abort = 0;
  const int64_t t_first = rank * kTile + warp * kLong;
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
  if (g.h0 != nullptr && on) state = two_floats(g.h0 + batch * g.dim + ch, 1);
  if (g.chunks > 1) cluster_wait();

  int buf = 0, s = 0;
  uint32_t parity = 0;
  bool alive = true;
  for (int64_t tile = 0, t0 = t_first; tile < stop; tile += stride, t0 += stride, buf ^= 1) {
    const int n = static_cast<int>(t0 >= stop ? 0 : min64(kLong, stop - t0));
    const uint32_t cut = __ballot_sync(0xffffffffu, flag != 0);
    flag = flag_of(t0 + stride);
    const bool plain = n == kLong && cut == 0;
    if (n > 0 && alive) {
      // A wait that runs out, as in Stream::wait.
      alive = sm100::mbar_wait(&full[warp][s], parity, &abort, &g_recurrence_error);
      if (!alive && lane == 0) {
        for (int i = 0, at = s, p = parity; i < kStages - (tile > 0 ? 1 : 0) && t0 + i * stride < stop; ++i) {
          sm100::mbar_drain(&full[warp][at], p);
          if (++at == kStages) {
            at = 0;
            p ^= 1;
          }
        }
      }
    }
    T *rows = stage(s);
    float2 a[kLong], b[kLong], p, h;
#pragma unroll
    for (int j = 0; j < kLong; ++j) {
      float2 c;
      gates2(stage_pair<T>(rows + j * kChan, lane), a[j], c);
      b[j] = mul2(c, stage_pair<T>(rows + (kLong + j) * kChan, lane));
    }
    scan_run<kLong>(a, b, n, cut, plain, p, h);
    const float2 in = tile_exchange(ex, buf, p, h, state, g.chunks, rank, reset != nullptr);
    auto save = [&](int j, float2 v) {
      if (g.saved != nullptr && on) put_two_floats(g.saved + (batch * g.runs + (t0 + j) / kRun) * g.dim + ch, v);
    };
    emit_run<kLong>(a, b, n, cut, plain, in, save,
                   [&](int j, float2 v) { store_pair<T, true>(rows + (kLong + j) * kChan + 2 * lane, v, true, true); });
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (n > 0 && alive) tma_store_3d(&maps.out_value, rows + kLong * kChan, ch0, static_cast<int>(t0), batch);
      sm100::bulk_commit();
      // The stage before this one has been read by its store: its next tile comes in.
      bulk_wait_read<1>();
      if (tile > 0 && alive) fetch(t0 + (kStages - 1) * stride, s == 0 ? kStages - 1 : s - 1);
    }
    if (++s == kStages) {
      s = 0;
      parity ^= 1;
    }
  }
  if (warp == 0 && rank == 0 && on) put_two_floats(g.h_last + batch * g.dim + ch, state);
  if (lane == 0) sm100::bulk_wait_read_all();
}

// Backward. With r_t = keep_t a_t ds_t the part of step t's gradient that reaches h_{t-1}:
//   ds_t = grad_t + r_{t+1},  grad_value = c ds,  grad_gate = a c (keep h_{t-1} - x) ds
// r is the forward's recurrence from the sequence's end, with the same P: a first pass over gate and
// grad for the segments' maps, then a second over all three with r coming in. h_{t-1} is scanned from
// the state saved before the run, in 32 bits; h itself is not read.
template <typename T, bool TMA, bool PAIRED, int PASS>
__global__ void __launch_bounds__(kThreads, TMA && sizeof(T) == 2 ? 3 : 2)
    recurrence_backward_kernel(const RecurrenceArgs g, const __grid_constant__ SequenceMaps maps) {
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ Exchange ex;
  __shared__ uint64_t full[kWarps][4];
  __shared__ int abort;
  using In = Stream<T, 3, TMA, PAIRED>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.x / g.chunks, chunk = blockIdx.x - unit * g.chunks;
  const int64_t batch = unit / g.channel_blocks;
  const int block = unit - static_cast<int>(batch) * g.channel_blocks;
  const Lane<PAIRED> at(block, g.dim);
  const bool graded = g.grad != nullptr;
  const uint32_t for_maps = graded ? 5u : 1u, for_all = graded ? 7u : 3u;  // gate, value, grad
  const uint8_t *reset = g.reset != nullptr ? g.reset + batch * g.steps : nullptr;
  const Items<false, PASS> items(g, chunk, warp);
  const int total = items.total, steps = static_cast<int>(g.steps);
  if (PASS == kBoth && g.chunks > 1) cluster_arrive();

  In in;
  if constexpr (TMA) {
    in.ring = reinterpret_cast<T *>(dynamic) + size_t(warp) * In::kDeep * 3 * kRun * kChan;
    in.full = full[warp];
    in.abort = &abort;
    in.maps[0] = &maps.gate;
    in.maps[1] = &maps.value;
    in.maps[2] = &maps.grad;
    in.ch0 = block * kChan;
    in.batch = static_cast<int>(batch);
    if (threadIdx.x == 0) abort = 0;
    if (lane == 0) {
#pragma unroll
      for (int s = 0; s < In::kDeep; ++s) sm100::mbar_init(&full[warp][s], 1);
      sm100::mbar_init_fence();
      sm100::fence_proxy_async_smem();
    }
    __syncthreads();
  } else {
    in.from[0] = static_cast<const T *>(g.gate) + batch * g.gate_batch + at.from;
    in.from[1] = static_cast<const T *>(g.value) + batch * g.value_batch + at.from;
    in.from[2] = static_cast<const T *>(g.grad) + (graded ? batch * g.steps * g.dim + at.from : 0);
    in.stride[0] = g.gate_step;
    in.stride[1] = g.value_step;
    in.stride[2] = g.dim;
    in.steps = steps;
    in.second = at.second;
  }
  auto which_of = [&](int i) { return PASS != kApply && i < items.count ? for_maps : for_all; };
  const int ahead = TMA ? In::kDeep : 1;
  for (int i = 0; i < ahead; ++i)
    if (i < total) in.fetch(items.start(i), which_of(i), i);
  uint32_t flag = total > 0 ? flag_of(reset, items.start(0), steps) : 0;
  int item = 0;
  auto flags = [&]() -> uint32_t {
    if (reset == nullptr) return 0;
    const uint32_t cut = __ballot_sync(0xffffffffu, flag != 0);
    flag = item + 1 < total ? flag_of(reset, items.start(item + 1), steps) : 0;
    return cut;
  };
  const float2 zero = make_float2(0.f, 0.f);
  float2 r = zero, p = make_float2(1.f, 1.f);
  uint32_t was_cut = 0;
  if (PASS != kApply) {
    for (; item < items.count; ++item) {
      const int t0 = items.start(item);
      const int n = min(kRun, steps - t0);
      const uint32_t cut = flags();
      in.wait(total - item);
      float2 a[kRun], gt[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        float2 c;
        gates2(in.get(0, j), a[j], c);
        gt[j] = graded ? in.get(2, j) : zero;
      }
      if constexpr (TMA) __syncwarp();  // all lanes have read the stage
      if (item + ahead < total) in.fetch(items.start(item + ahead), which_of(item + ahead), 0);
      in.next();
      if (n == kRun && cut == 0) {
#pragma unroll
        for (int j = kRun - 1; j >= 0; --j) {
          r = mul2(a[j], add2(gt[j], r));
          p = mul2(p, a[j]);
        }
      } else {
#pragma unroll
        for (int j = kRun - 1; j >= 0; --j) {
          if (j < n) {
            r = mul2(a[j], add2(gt[j], r));
            p = mul2(p, a[j]);
            if ((cut >> j) & 1u) r = zero;
          }
        }
        was_cut |= cut;
      }
    }
    if (was_cut != 0) p = both(kCut);
  }
  float2 back = zero;  // r of the step after the sequence
  if (g.grad_last != nullptr) back = two_floats(g.grad_last + batch * g.dim + at.from, at.second);
  if (PASS == kBoth && g.chunks > 1) cluster_wait();  // all have started
  back = exchange<false, PAIRED, PASS>(g, batch, at, chunk, p, r, back, ex);
  if (PASS == kMaps) return;

  T *grad_gate = static_cast<T *>(g.grad_gate) + batch * g.steps * g.dim + at.ch;
  T *grad_value = static_cast<T *>(g.grad_value) + batch * g.steps * g.dim + at.ch;
  auto before_of = [&](int i) -> float2 {
    if (i >= total) return zero;
    return two_floats(g.saved + (batch * g.runs + items.start(i) / kRun) * g.dim + at.from, at.second);
  };
  float2 before = before_of(item);
  for (; item < total; ++item) {
    const int t0 = items.start(item);
    const int n = min(kRun, steps - t0);
    const uint32_t cut = flags();
    float2 h = before;
    before = before_of(item + 1);
    in.wait(total - item);
    float2 a[kRun], c[kRun], u[kRun], gt[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      gates2(in.get(0, j), a[j], c[j]);
      u[j] = in.get(1, j);
      if constexpr (!TMA) gt[j] = graded ? in.get(2, j) : zero;
    }
    if constexpr (!TMA)
      if (item + 1 < total) in.fetch(items.start(item + 1), for_all, 0);
    auto grad_at = [&](int j) -> float2 {
      if constexpr (TMA) return graded ? in.get(2, j) : zero;
      else return gt[j];
    };
    auto put = [&](int j, float2 ds) {
      const float2 gx = mul2(c[j], ds), gf = mul2(mul2(a[j], gx), u[j]);
      if constexpr (TMA) {
        store_pair<T, true>(in.rows(0) + j * kChan + 2 * lane, gf, true, true);
        store_pair<T, true>(in.rows(1) + j * kChan + 2 * lane, gx, true, true);
      } else {
        store_pair<T, PAIRED>(grad_gate + int64_t(t0 + j) * g.dim, gf, at.on0, at.on1);
        store_pair<T, PAIRED>(grad_value + int64_t(t0 + j) * g.dim, gx, at.on0, at.on1);
      }
    };
    const float2 minus = make_float2(-1.f, -1.f);
    if (n == kRun && cut == 0) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const float2 x = u[j];
        u[j] = fma2(x, minus, h);  // keep h_{t-1} - x
        h = fma2(a[j], h, mul2(c[j], x));
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        const float2 ds = add2(grad_at(j), back);
        back = mul2(a[j], ds);
        put(j, ds);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (j < n) {
          const float2 x = u[j];
          if ((cut >> j) & 1u) h = zero;
          u[j] = fma2(x, minus, h);
          h = fma2(a[j], h, mul2(c[j], x));
        }
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        if (j < n) {
          const float2 ds = add2(grad_at(j), back);
          back = mul2(a[j], ds);
          put(j, ds);
          if ((cut >> j) & 1u) back = zero;
        }
      }
    }
    if constexpr (TMA) {
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (in.alive) {
          tma_store_3d(&maps.out_gate, in.rows(0), in.ch0, t0, in.batch);
          tma_store_3d(&maps.out_value, in.rows(1), in.ch0, t0, in.batch);
        }
        sm100::bulk_commit();
        bulk_wait_read<1>();  // the stage before this one has been read by its stores
      }
      // That stage's next run comes in; the first run's stage has no store before it.
      if (in.stored && item - 1 + In::kDeep < total) in.fetch(items.start(item - 1 + In::kDeep), for_all, In::kDeep - 1);
      in.stored = true;
    }
    in.next();
  }
  if (warp == 0 && chunk == 0 && g.grad_h0 != nullptr) {
    float *out = g.grad_h0 + batch * g.dim + at.ch;
    if (at.on0) out[0] = back.x;
    if (at.on1) out[kSecond<PAIRED>] = back.y;
  }
  if (TMA && lane == 0) sm100::bulk_wait_read_all();
}

// One token of every row: state (f32, updated in place) and h. One read and one write of each operand:
// launch latency up to some hundred rows (8 x 1024 bf16 1.2 us), then HBM. N channels a thread: 4 where
// addresses and strides allow it, else 1 (4096 x 4096 bf16: 36 us, 6.6 TB/s, and 61 us).
template <typename T, int N>
__global__ void __launch_bounds__(256) recurrence_step_kernel(const T *__restrict__ gate, int64_t gate_row,
                                                              const T *__restrict__ value, int64_t value_row,
                                                              const uint8_t *__restrict__ reset, int64_t dim,
                                                              float *state, int64_t state_row, T *__restrict__ h) {
  struct alignas(N * sizeof(T)) Values {
    T v[N];
  };
  struct alignas(N * sizeof(float)) States {
    float v[N];
  };
  const int64_t ch = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) * N;
  const int64_t row = blockIdx.y;
  if (ch >= dim) return;
  const Values f = *reinterpret_cast<const Values *>(gate + row * gate_row + ch);
  const Values x = *reinterpret_cast<const Values *>(value + row * value_row + ch);
  States s = *reinterpret_cast<const States *>(state + row * state_row + ch);
  const bool fresh = reset != nullptr && reset[row] != 0;
  Values out;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const int j = N > 1 ? i + 1 : i;
    float2 a, c;
    gates2(make_float2(to_f32<T>(f.v[i]), N > 1 ? to_f32<T>(f.v[j]) : 0.f), a, c);
    s.v[i] = fmaf(a.x, fresh ? 0.f : s.v[i], c.x * to_f32<T>(x.v[i]));
    out.v[i] = from_f32<T>(s.v[i]);
    if (N > 1) {
      s.v[j] = fmaf(a.y, fresh ? 0.f : s.v[j], c.y * to_f32<T>(x.v[j]));
      out.v[j] = from_f32<T>(s.v[j]);
    }
  }
  *reinterpret_cast<States *>(state + row * state_row + ch) = s;
  *reinterpret_cast<Values *>(h + row * dim + ch) = out;
}

inline size_t elem_bytes(int dtype) { return dtype == TROPNN_B200_F32 ? 4 : 2; }
inline bool paired(const void *p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (2 * elem_bytes(dtype)) == 0; }

// Blocks of channels of all rows, by 8 chunks each, below 2^31: tested so that nothing overflows.
bool fits_grid(int64_t batch, int64_t dim) {
  const int64_t most = 0x7fffffffLL / kMaxCluster;
  return dim <= most * kChan && (batch == 0 || ceil_div(dim, kChan) <= most / batch);
}
int check_sizes(const char *what, int dtype, int64_t batch, int64_t steps, int64_t dim) {
  TB_REQUIRE(is_float_dtype(dtype), TROPNN_B200_ERR_DTYPE, "%s: dtype %d is not f32/f16/bf16", what, dtype);
  TB_REQUIRE(batch >= 0 && steps >= 0 && dim >= 0, TROPNN_B200_ERR_INVALID, "%s: bad sizes (batch %lld, steps %lld, dim %lld)",
             what, (long long)batch, (long long)steps, (long long)dim);
  TB_REQUIRE(fits_grid(batch, dim), TROPNN_B200_ERR_INVALID, "%s: batch x dim too large", what);
  TB_REQUIRE(steps <= 0x7fffffffLL - kRun, TROPNN_B200_ERR_INVALID, "%s: %lld steps are too many", what, (long long)steps);
  return TROPNN_B200_OK;
}

// How a sequence is shared out: chunks of kWarps segments, a CTA each, as many as are on the GPU at once.
// Up to 8 chunks are a cluster. Where 8 are less than half of that, and at least 4 runs a segment are
// left, there are more chunks and two launches; a forward pass not cut so goes by tiles. 1 x 16384 x 1024
// bf16, cut and not: forward 39 and 58 us, backward 45 and 82 us.
struct Plan {
  int chunks = 1;
  bool two_launches = false;
  int64_t segment_runs = 0;
};
Plan plan_for(int64_t units, int64_t runs, int64_t slots) {
  Plan p;
  p.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxCluster, slots / units, runs / kWarps})));
  if (p.chunks == kMaxCluster && units * p.chunks * 2 <= slots) {
    const int64_t many = min64(slots / units, runs / (4 * kWarps));
    if (many >= 2 * kMaxCluster) {
      p.chunks = static_cast<int>(many);
      p.two_launches = true;
    }
  }
  p.segment_runs = std::max<int64_t>(1, ceil_div(runs, int64_t(p.chunks) * kWarps));
  if (p.two_launches) p.chunks = static_cast<int>(ceil_div(runs, p.segment_runs * kWarps));
  return p;
}
int64_t units_of(int64_t batch, int64_t dim) { return batch * ceil_div(dim, kChan); }
// CTAs on the GPU at once. The SMs are a constant: the workspace query must not need a device.
constexpr int kSms = 148;
int64_t slots_of(bool forward, int dtype) { return kSms * (dtype == TROPNN_B200_F32 || !forward ? 2 : 3); }
size_t maps_bytes(const Plan &p, int64_t batch, int64_t dim) {
  return p.two_launches ? static_cast<size_t>(batch * p.chunks * kMapSlots * dim) * sizeof(float2) : 0;
}

// Sequences come by TMA where they can, else by loads of pairs of channels, else of single ones. 8 x 2048 x
// 1024 bf16 by TMA and by pairs: forward 29.0 and 30.5 us, backward 44 and 59; 1 x 65536 x 256 f16 37 and
// 54, 45 and 56.
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

int launch_clusters(const char *what, const void *kernel, size_t smem, int64_t ctas, int cluster, RecurrenceArgs &g,
                    SequenceMaps &maps, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(ctas));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  // The static part counts too: above 48 KB in all the kernel has to be told.
  if (smem > 0) TB_CHECK(ensure_dynamic_smem(kernel, std::max<size_t>(smem, 49 * 1024), what));
  void *args[] = {&g, &maps};
  cudaLaunchKernelExC(&config, kernel, args);
  return check_launch(what);
}
template <bool FORWARD, typename T, bool TMA, bool PAIRED, int PASS>
int launch_pass(const char *what, RecurrenceArgs g, SequenceMaps &maps, int64_t units, cudaStream_t stream) {
  const void *kernel;
  if constexpr (FORWARD) kernel = reinterpret_cast<const void *>(recurrence_forward_kernel<T, TMA, PAIRED, PASS>);
  else kernel = reinterpret_cast<const void *>(recurrence_backward_kernel<T, TMA, PAIRED, PASS>);
  return launch_clusters(what, kernel, TMA ? kRingBytes<T, FORWARD ? 2 : 3> : 0, units * g.chunks, PASS == kBoth ? g.chunks : 1, g,
                         maps, stream);
}
template <typename T, bool TMA, bool PAIRED>
int launch_tiles(const char *what, RecurrenceArgs g, SequenceMaps &maps, int64_t units, cudaStream_t stream) {
  const int64_t tiles = ceil_div(g.steps, kWarps * kTileRun<T>);
  g.chunks = 1;  // CTAs of a cluster, two of them an SM in all
  while (g.chunks < kMaxCluster && units * g.chunks * 2 <= 2 * kSms && g.chunks * 2 <= tiles) g.chunks *= 2;
  const void *kernel = TMA ? reinterpret_cast<const void *>(recurrence_tiles_tma_kernel<T>)
                           : reinterpret_cast<const void *>(recurrence_tiles_kernel<T, PAIRED>);
  return launch_clusters(what, kernel, TMA ? kTileRingBytes<T> : 0, units * g.chunks, g.chunks, g, maps, stream);
}
template <bool FORWARD, typename T, bool TMA, bool PAIRED>
int launch_form(const char *what, const RecurrenceArgs &g, SequenceMaps &maps, int64_t units, bool two_launches, cudaStream_t stream) {
  if (!two_launches) {
    if constexpr (FORWARD) return launch_tiles<T, TMA, PAIRED>(what, g, maps, units, stream);
    else return launch_pass<FORWARD, T, TMA, PAIRED, kBoth>(what, g, maps, units, stream);
  }
  TB_CHECK((launch_pass<FORWARD, T, TMA, PAIRED, kMaps>(what, g, maps, units, stream)));
  return launch_pass<FORWARD, T, TMA, PAIRED, kApply>(what, g, maps, units, stream);
}
template <bool FORWARD, typename T>
int launch_typed(const char *what, const RecurrenceArgs &g, int dtype, int64_t batch, bool pair, bool two_launches, cudaStream_t stream) {
  const int64_t units = batch * g.channel_blocks, steps = g.steps, dim = g.dim;
  const int run = FORWARD && !two_launches ? kTileRun<T> : kRun;
  SequenceMaps maps{};
  bool fits = pair && steps > 0 && sequence_map(&maps.gate, g.gate, dtype, batch, steps, dim, g.gate_batch, g.gate_step, run) &&
              sequence_map(&maps.value, g.value, dtype, batch, steps, dim, g.value_batch, g.value_step, run);
  if (FORWARD) {
    fits = fits && sequence_map(&maps.out_value, g.h, dtype, batch, steps, dim, steps * dim, dim, run);
  } else {
    fits = fits && (g.grad == nullptr || sequence_map(&maps.grad, g.grad, dtype, batch, steps, dim, steps * dim, dim, run)) &&
           sequence_map(&maps.out_gate, g.grad_gate, dtype, batch, steps, dim, steps * dim, dim, run) &&
           sequence_map(&maps.out_value, g.grad_value, dtype, batch, steps, dim, steps * dim, dim, run);
  }
  if (fits) return launch_form<FORWARD, T, true, true>(what, g, maps, units, two_launches, stream);
  if (pair) return launch_form<FORWARD, T, false, true>(what, g, maps, units, two_launches, stream);
  return launch_form<FORWARD, T, false, false>(what, g, maps, units, two_launches, stream);
}

template <bool FORWARD>
int launch_recurrence(const char *what, RecurrenceArgs g, int dtype, int64_t batch, bool pair, void *workspace,
                      size_t workspace_bytes, cudaStream_t stream) {
  const Plan plan = plan_for(batch * g.channel_blocks, g.runs, slots_of(FORWARD, dtype));
  const size_t need = maps_bytes(plan, batch, g.dim);
  TB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), TROPNN_B200_ERR_WORKSPACE,
             "%s: %zu bytes of workspace, %zu needed", what, workspace_bytes, need);
  g.chunks = plan.chunks;
  g.segment_runs = plan.segment_runs;
  g.maps = static_cast<float2 *>(workspace);
  if (dtype == TROPNN_B200_F32) return launch_typed<FORWARD, float>(what, g, dtype, batch, pair, plan.two_launches, stream);
  if (dtype == TROPNN_B200_F16) return launch_typed<FORWARD, __half>(what, g, dtype, batch, pair, plan.two_launches, stream);
  return launch_typed<FORWARD, __nv_bfloat16>(what, g, dtype, batch, pair, plan.two_launches, stream);
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
  if (batch <= 0 || steps <= 0 || dim <= 0 || !fits_grid(batch, dim)) return 0;
  return static_cast<size_t>(batch * ceil_div(steps, kRun) * dim) * sizeof(float);
}

size_t tropnn_b200_recurrence_workspace_size(int64_t batch, int64_t steps, int64_t dim, int dtype) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || !is_float_dtype(dtype) || !fits_grid(batch, dim)) return 0;
  const int64_t units = units_of(batch, dim), runs = ceil_div(steps, kRun);
  return std::max(maps_bytes(plan_for(units, runs, slots_of(true, dtype)), batch, dim),
                  maps_bytes(plan_for(units, runs, slots_of(false, dtype)), batch, dim));
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
  g.runs = ceil_div(steps, kRun);
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
  g.runs = ceil_div(steps, kRun);
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
    const size_t eb = elem_bytes(dtype);
    const char *gp = static_cast<const char *>(gate) + done * gate_stride * int64_t(eb);
    const char *vp = static_cast<const char *>(value) + done * value_stride * int64_t(eb);
    char *hp = static_cast<char *>(h) + done * dim * int64_t(eb);
    const uint8_t *rp = reset != nullptr ? reset + done : nullptr;
    float *sp = state + done * state_stride;
    const bool wide = (dim | gate_stride | value_stride | state_stride) % 4 == 0 &&
                      (reinterpret_cast<uintptr_t>(gp) | reinterpret_cast<uintptr_t>(vp) | reinterpret_cast<uintptr_t>(hp)) % (4 * eb) == 0 &&
                      reinterpret_cast<uintptr_t>(sp) % 16 == 0;
    const int64_t threads = wide ? dim / 4 : dim;
    const dim3 grid(static_cast<unsigned>(ceil_div(threads, 256)), static_cast<unsigned>(rows));
#define TB_STEP_N(T, N)                                                                                          \
  recurrence_step_kernel<T, N><<<grid, 256, 0, as_stream(stream)>>>(reinterpret_cast<const T *>(gp), gate_stride, \
                                                                    reinterpret_cast<const T *>(vp), value_stride, rp, \
                                                                    dim, sp, state_stride, reinterpret_cast<T *>(hp))
#define TB_STEP(T) wide ? (TB_STEP_N(T, 4)) : (TB_STEP_N(T, 1))
    if (dtype == TROPNN_B200_F32) TB_STEP(float);
    else if (dtype == TROPNN_B200_F16) TB_STEP(__half);
    else TB_STEP(__nv_bfloat16);
#undef TB_STEP_N
#undef TB_STEP
    TB_CHECK(check_launch(what));
    done += rows;
  }
  return clear_error();
}

}  // extern "C"
