// Beam search selection: the best tokens of each beam, then the best beams x
// tokens of each batch element, in one launch.
//
// The bound is one read of the logits. A row is cut into slices, one CTA
// each, so that a few rows still occupy many SMs; a CTA reads its slice once,
// in tiles held in registers, and keeps a running (max, sum) per thread and
// the slice's `beams` best keys. A tile's candidates are found by a threshold
// that is a lower bound of its beams-th best value: for the first tile from
// the sorted lane maxima of the warps, later the beams-th best of the tiles
// so far, taken again whenever their number has doubled. (Without that step,
// with some 17 candidates a tile in the place of 8 / tile, 64 x 8 beams take
// 31 us in the place of 21; with it once, after the first tile, 32 x 16 beams
// over 95,351 take 157 us in the place of 45, for their candidates no longer
// fit.) They are collected without a barrier. At the end those that reach the
// last bar are put in order by their ranks, counted, each against all. Keys
// are (logit, token) pairs as 64-bit integers, all different, so the order is
// total and independent of the order in which threads append.
//
// The last CTA of a batch element to arrive joins the slices: a warp takes a
// beam, whose slices' sorted lists are merged by shuffles (up to eight beams:
// a lane per slice, the best of their heads once per rank, since there may be
// 32 lists), and merges it with its other beams' offers; then the warps'.
// (Once per rank throughout: 1 x 32 beams over 4,096 tokens 26 us, merged 11.)
//
// Measured (B200): 4 beams over 32,000 fp32 logits 6.3 us; 64 x 8 beams, 15% of
// them finished and not read, 20.6 us = 2.7 TB/s; 32 x 32 beams 51 us: a row's CTA spends half
// its time outside the tiles (threshold, ranks, arrival and join), and with
// three or four rows on an SM that is not all hidden. More slices only
// multiply it (two 24 us, four 32 us), loads two tiles ahead change nothing.
#include <float.h>

#include <algorithm>

#include "paged.cuh"

namespace ce {
namespace paged {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kMaxGroups = 16384;  // batch elements: arrival counters at the front of the workspace
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kElems = 16;         // logits per thread and tile
// Epochs of a slice: the first tile, then 2, 4, 8, 16, 32 tiles, then the rest.
constexpr int kEpochs = 7;
constexpr int kFirst = 512;        // candidates of the first epoch
constexpr int kLater = 640;        // of each later one: warps may run eight tiles ahead of a bar
constexpr int kKept = 512;         // candidates that are ranked
constexpr int kListKeys = 256;     // keys of one beam's lists at the join: slices x beams

struct BeamArgs {
  float *scores_out;
  int32_t *parents, *tokens;
  uint8_t *finished_out;
  const void *logits;
  long long ld;
  const float *scores;
  const uint8_t *finished;
  int batch, beams, vocab, eos, pad, slices;
  int *arrivals;             // [batch], zero between calls
  unsigned long long *best;  // [rows][slices][beams], 0: none
  float2 *sums;              // [rows][slices]: max, sum of e^(x - max)
};

constexpr float kLog2e = 1.44269504088896341f;

// A logit as the selection takes it: NaN is -inf, +inf the largest finite
// value, -0 is +0.
template <typename T>
__device__ __forceinline__ float logit_of(T v) {
  const float x = to_float(v);
  return fminf(fmaxf(x, -INFINITY), FLT_MAX) + 0.f;  // fmaxf gives the number where the other is NaN
}

// Keys order tokens by (logit descending, token ascending) as integers.
__device__ __forceinline__ unsigned long long key_of(float x, int token) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 is +0
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((unsigned long long)o << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_token(unsigned long long k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The warp's 32 values in descending order of lanes.
__device__ __forceinline__ float warp_sorted(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step; step >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, v, step);
      const bool up = ((lane & step) != 0) == ((lane & size) != 0);  // this lane keeps the larger one
      v = up ? fmaxf(v, y) : fminf(v, y);
    }
  return v;
}

// The 32 largest of two lists, in descending order of lanes: `a` in that order,
// `b` in the opposite one. Their lane maxima are those 32, first rising, then
// falling or a turn of it, which five steps sort.
template <typename T>
__device__ __forceinline__ T warp_merged(T a, T b) {
  const int lane = threadIdx.x & 31;
  T v = a > b ? a : b;
#pragma unroll
  for (int step = 16; step; step >>= 1) {
    const T y = __shfl_xor_sync(0xffffffffu, v, step);
    v = (lane & step ? y < v : y > v) ? y : v;
  }
  return v;
}

// Joins (max, sum of e^(x - max)) pairs.
__device__ __forceinline__ void add_sum(float &m, float &l, float m1, float l1) {
  if (m1 > m) {
    const float x = m;
    m = m1, m1 = x;
    const float y = l;
    l = l1, l1 = y;
  }
  if (m1 != -INFINITY) l += l1 * exp2_approx((m1 - m) * kLog2e);
}

struct Shared {
  unsigned long long buffer[kFirst + (kEpochs - 1) * kLater];  // candidates; at the join the lists, per warp
  unsigned long long top[kMaxBeams];
  float2 kth[kWarps];
  float2 sums[kWarps];
  unsigned long long round[kWarps];
  unsigned long long kept[kKept];  // candidates not below the last bar; at the join 32 per warp
  int token[kMaxBeams][kMaxBeams];  // [beam][rank]
  int count[kEpochs], passed[kEpochs];  // candidates; warps past the epoch
  int keep, last;
  float best[32];                  // of the epochs that all warps have passed, sorted
  float bar;                       // what a later tile's candidates exceed
};
static_assert(kFirst + (kEpochs - 1) * kLater >= kWarps * kListKeys && kFirst >= 3 * kMaxBeams, "the lists of the join");
static_assert(kKept >= 32 * kWarps, "a list per warp");
static_assert(kElems == 16, "four tops of four");

// The `beams` best keys of the slice's tokens [t0, t1) by taking the best that
// is below the last taken, once per rank, from memory: for slices where too
// many values pass the threshold (equal or ascending logits).
template <typename T>
__device__ __noinline__ void take_in_rounds(Shared &sh, const T *x, int t0, int t1, int beams) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long last = ~0ull;
  for (int r = 0; r < beams; ++r) {
    unsigned long long k = 0;
    for (int i = t0 + (int)threadIdx.x; i < t1; i += kThreads) {
      const unsigned long long c = key_of(logit_of(x[i]), i);
      k = c < last && c > k ? c : k;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long y = __shfl_xor_sync(0xffffffffu, k, o);
      k = y > k ? y : k;
    }
    if (lane == 0) sh.round[warp] = k;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) k = sh.round[w] > k ? sh.round[w] : k;
    __syncthreads();
    if (threadIdx.x == 0) sh.top[r] = k;  // 0: no more
    last = k;
  }
  __syncthreads();
}

__device__ __forceinline__ int epoch_start(int epoch) { return epoch == 0 ? 0 : kFirst + (epoch - 1) * kLater; }
__device__ __forceinline__ int epoch_size(int epoch) { return epoch == 0 ? kFirst : kLater; }

// The `beams` best of n keys, in order, by their ranks among all; 0 past the last.
__device__ __forceinline__ void rank_candidates(Shared &sh, const unsigned long long *keys, int n, int beams) {
  if ((int)threadIdx.x < beams) sh.top[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long k = keys[i];
    int rank = 0;
    for (int q = 0; q < n; ++q) rank += keys[q] > k;
    if (rank < beams) sh.top[rank] = k;
  }
  __syncthreads();
}

// By one warp, when all have passed an epoch: takes its candidates into the 32
// best logits so far and returns the beams-th (-inf if there are fewer).
__device__ __forceinline__ float later_bar(Shared &sh, int epoch, int beams) {
  const int lane = threadIdx.x & 31, n = *(volatile int *)&sh.count[epoch];
  if (n > epoch_size(epoch)) return INFINITY;  // too many: the rounds decide
  float best = epoch == 0 ? -INFINITY : *(volatile float *)&sh.best[lane];
  for (int i = lane; i - lane < n; i += 32) {
    const float v = i < n ? key_logit(sh.buffer[epoch_start(epoch) + i]) : -INFINITY;
    const float least = __shfl_sync(0xffffffffu, best, 31);
    if (!__any_sync(0xffffffffu, v > least)) continue;
    best = warp_merged(best, __shfl_sync(0xffffffffu, warp_sorted(v), 31 - lane));
  }
  *(volatile float *)&sh.best[lane] = best;
  return __shfl_sync(0xffffffffu, best, beams - 1);
}

// The largest float below a finite x (so that y > it means y >= x).
__device__ __forceinline__ float just_below(float x) {
  const int b = __float_as_int(x);
  return x == 0.f ? -__int_as_float(1) : __int_as_float(x > 0.f ? b - 1 : b + 1);
}

// The sum of e^(x - base) over N values, none above a finite base: one
// multiply-add and one 2^y a value, relative to the rounded base log2 e, whose
// rounding is taken back at the end.
template <int N>
__device__ __forceinline__ float sum_exp(const float (&x)[N], float base) {
  const float b = base * kLog2e;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    s0 += exp2_approx(fmaf(x[i], kLog2e, -b));
    s1 += exp2_approx(fmaf(x[i + 1], kLog2e, -b));
  }
  return (s0 + s1) * exp2_approx(-fmaf(base, kLog2e, -b));
}

// open: the batch element's unfinished beams, read behind the first loads.
template <typename T>
__device__ __forceinline__ bool slice_of_row(const BeamArgs &a, Shared &sh, int group, int beam, int slice, uint32_t &open) {
  constexpr int kPerVec = 16 / sizeof(T), kVecs = kElems / kPerVec, kTile = kThreads * kVecs;  // in vectors
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams;
  const int row = group * K + beam;
  const T *x = static_cast<const T *>(a.logits) + row * a.ld;
  // 16-byte vectors of the row from its first aligned element on; the few
  // elements before and after them go to the first and last slice, one per thread
  const int head = min(a.vocab, (int)((16u - (unsigned)(reinterpret_cast<uintptr_t>(x) & 15u)) % 16u / sizeof(T)));
  const int vecs = (a.vocab - head) / kPerVec, tail = a.vocab - head - vecs * kPerVec;
  const int per = (vecs + a.slices - 1) / a.slices;
  const int v0 = min(vecs, slice * per), v1 = min(vecs, v0 + per);
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
  int extra = -1;  // token of this thread's single element
  if (slice == 0 && tid < head) extra = tid;
  if (slice == a.slices - 1 && tid >= 128 && tid < 128 + tail) extra = a.vocab - tail + tid - 128;

  uint4 raw[kVecs];
  auto load = [&](int at) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      if (at + v * kThreads < v1) raw[v] = __ldcs(xv + at + v * kThreads);
  };
  load(v0 + tid);
  open = __ballot_sync(0xffffffffu, lane < K && !a.finished[group * K + min(lane, K - 1)]);
  if (!(open >> beam & 1)) return false;
  float ex = extra >= 0 ? logit_of(x[extra]) : -INFINITY;
  float m = ex, l = ex > -INFINITY ? 1.f : 0.f;
  if (tid < kEpochs) sh.count[tid] = sh.passed[tid] = 0;
  if (tid == 0) sh.keep = 0, sh.bar = -INFINITY;
  float bar = -INFINITY;
  const int tiles = max(1, (v1 - v0 + kTile - 1) / kTile);
  for (int tile = 0; tile < tiles; ++tile) {
    float e[kElems];
    const int at = v0 + tile * kTile + tid;
    const bool whole = v0 + (tile + 1) * kTile <= v1;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const T *p = reinterpret_cast<const T *>(&raw[v]);
#pragma unroll
      for (int i = 0; i < kPerVec; ++i) e[v * kPerVec + i] = to_float(p[i]);
    }
    if (!whole) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
        if (at + v * kThreads >= v1)
#pragma unroll
          for (int i = 0; i < kPerVec; ++i) e[v * kPerVec + i] = -INFINITY;
    }
    if (tile + 1 < tiles) load(at + kTile);  // under way during this tile
    float tops[kElems / 4];  // of four numbers each: a NaN is passed over
#pragma unroll
    for (int i = 0; i < kElems; i += 4) tops[i / 4] = fmaxf(fmaxf(e[i], e[i + 1]), fmaxf(e[i + 2], e[i + 3]));
    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (!(top <= -INFINITY)) {
      float base = fmaxf(top, m), s = sum_exp(e, base);
      // a NaN, +inf, or values so large that the rounding of their product with
      // log2 e is no small number (from 2^30 on its 2^y can be 0 or infinite)
      if (!(s <= kElems * 1.001f) || fabsf(base) > 1048576.f) {
        top = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
          e[i] = logit_of(e[i]);
          tops[i / 4] = i % 4 ? fmaxf(tops[i / 4], e[i]) : e[i];
          top = fmaxf(top, e[i]);
        }
        base = fmaxf(top, m);
        if (base > -INFINITY)
#pragma unroll
          for (int i = 0; i < kElems; ++i) s += exp2_approx((e[i] - base) * kLog2e);  // a difference cannot overflow upwards
      }
      if (base > -INFINITY) l = l * exp2_approx((m - base) * kLog2e) + s, m = base;
    }
    // candidates: values above `bar`
    if (tile == 0) {
      if (extra < head) top = fmaxf(top, ex);
      // At least K of the block's lane maxima reach the K-th of any warp, and
      // as many reach the ceil(K / 8)-th of every one of the 8 warps.
      const float sorted = warp_sorted(top), few = __shfl_sync(0xffffffffu, sorted, (K + kWarps - 1) / kWarps - 1),
                  kth = __shfl_sync(0xffffffffu, sorted, K - 1);
      if (lane == 0) sh.kth[warp] = make_float2(few, kth);
      __syncthreads();
      float every = sh.kth[0].x;
      bar = sh.kth[0].y;
      for (int w = 1; w < kWarps; ++w) every = fminf(every, sh.kth[w].x), bar = fmaxf(bar, sh.kth[w].y);
      bar = fmaxf(bar, every);
      if (bar > -INFINITY) bar = just_below(bar);
    } else {
      bar = fmaxf(bar, *(volatile float *)&sh.bar);
    }
    const int epoch = min(31 - __clz(tile + 1), kEpochs - 1);
    auto offer = [&](int to, float y, int token) {
      const int n = atomicAdd(&sh.count[to], 1);
      if (n < epoch_size(to)) sh.buffer[epoch_start(to) + n] = key_of(y, token);
    };
    if (top > bar) {
#pragma unroll
      for (int i = 0; i < kElems; i += 4)  // four at a time: hardly any of them has one
        if (tops[i / 4] > bar) {
#pragma unroll
          for (int y = i; y < i + 4; ++y)
            if (e[y] > bar) offer(epoch, e[y], head + (at + y / kPerVec * kThreads) * kPerVec + y % kPerVec);
        }
    }
    // the row's last elements, behind all tiles by their tokens, count with the last epoch
    if (tile == 0 && ex > bar) offer(extra < head ? 0 : kEpochs - 1, ex, extra);
    if (tile + 1 < tiles && epoch < kEpochs - 1 && tile == (2 << epoch) - 2) {
      // The last warp to have offered its part of the epoch takes the K-th
      // best so far as the later tiles' bar; nobody waits for it. (An equal
      // value of a later token is no better.) So each epoch, with as many
      // tiles as all before it, has about K candidates.
      __syncwarp();
      int passed = 0;
      if (lane == 0) {
        __threadfence_block();
        passed = atomicAdd(&sh.passed[epoch], 1);
        __threadfence_block();
      }
      passed = __shfl_sync(0xffffffffu, passed, 0);
      __syncwarp();
      if (passed == kWarps - 1) {
        const float kth = later_bar(sh, epoch, K);
        if (lane == 0) *(volatile float *)&sh.bar = kth;
      }
    }
  }
  __syncthreads();
  const int t0 = slice == 0 ? 0 : head + v0 * kPerVec, t1 = slice == a.slices - 1 ? a.vocab : head + v1 * kPerVec;
  int n = 0, first = sh.count[0];
  bool over = false;
#pragma unroll
  for (int i = 0; i < kEpochs; ++i) n += sh.count[i], over |= sh.count[i] > epoch_size(i);
  if (!over && n < K) {
    // Fewer than K values are finite: tokens of logit -inf follow, the
    // lowest first. K of them, or all, stand among the first 2 K tokens.
    __syncthreads();
    if (tid < min(2 * K, t1 - t0) && logit_of(x[t0 + tid]) == -INFINITY)
      sh.buffer[atomicAdd(&sh.count[0], 1)] = key_of(-INFINITY, t0 + tid);
    __syncthreads();
    n += sh.count[0] - first;
    first = sh.count[0];
  }
  const unsigned long long *keys = sh.buffer;
  if (!over && n > first) {  // those that reach the last bar, together
    const float least = sh.bar;
#pragma unroll 1
    for (int i = 0; i < kEpochs; ++i)
      for (int c = tid; c < sh.count[i]; c += kThreads) {
        const unsigned long long k = sh.buffer[epoch_start(i) + c];
        if (key_logit(k) >= least) {
          const int to = atomicAdd(&sh.keep, 1);
          if (to < kKept) sh.kept[to] = k;
        }
      }
    __syncthreads();
    keys = sh.kept, n = sh.keep, over = n > kKept;
  }
  if (over) take_in_rounds(sh, x, t0, t1, K);
  else rank_candidates(sh, keys, n, K);
#pragma unroll
  for (int o = 16; o; o >>= 1) add_sum(m, l, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o));
  if (lane == 0) sh.sums[warp] = make_float2(m, l);
  __syncthreads();
  const size_t list = (size_t)row * a.slices + slice;
  if (tid < K) __stcg(a.best + list * K + tid, sh.top[tid]);
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) add_sum(m, l, sh.sums[w].x, sh.sums[w].y);
    __stcg(a.sums + list, make_float2(m, l));
  }
  return true;
}

// The best key of the warp's lanes, and which lane holds it (keys differ).
__device__ __forceinline__ bool warp_best(unsigned long long k) {
  const uint32_t hi = (uint32_t)(k >> 32), top = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t lo = hi == top ? (uint32_t)k : 0u;
  const uint32_t low = __reduce_max_sync(0xffffffffu, lo);
  return hi == top && lo == low && k != 0;
}

// The offers of one beam, best first by lanes, from the sorted lists of its
// slices: keys of score, beam and rank; 0 past the last.
__device__ __forceinline__ unsigned long long offers_of_row(const BeamArgs &a, Shared &sh, int group, int beam) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = a.beams;
  const size_t row = (size_t)group * K + beam;
  const float base = a.scores[row];
  if (a.finished[row]) {
    if (lane == 0) sh.token[beam][0] = a.pad;
    return lane == 0 ? key_of(base != base ? -INFINITY : base, beam * 32) : 0ull;
  }
  unsigned long long *lists = sh.buffer + warp * kListKeys, top;
  for (int i = lane; i < a.slices * K; i += 32) lists[i] = __ldcg(a.best + row * a.slices * K + i);
  float m = -INFINITY, l = 0.f;
  if (lane < a.slices) {
    const float2 p = __ldcg(a.sums + row * a.slices + lane);
    m = p.x, l = p.y;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) add_sum(m, l, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o));
  const float lse = m + logf(l);
  __syncwarp();
  if (K <= 8 && a.slices > 1) {  // few ranks, up to 32 lists: a lane per slice, the best of their heads once per rank
    unsigned long long *taken = sh.kept + warp * 32;
    taken[lane] = 0;
    __syncwarp();
    int at = 0;
    for (int r = 0; r < min(K, a.vocab); ++r) {
      const unsigned long long k = lane < a.slices && at < K ? lists[lane * K + at] : 0ull;
      if (warp_best(k)) taken[r] = k, ++at;
    }
    __syncwarp();
    top = taken[lane];
  } else {
    unsigned long long t[8];  // the odd ones in the opposite order
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = i % 2 ? 31 - lane : lane;
      t[i] = i < a.slices && at < K ? lists[i * K + at] : 0ull;
    }
#pragma unroll
    for (int step = 1; step < 8; step *= 2)  // merges of a round side by side
      if (step < a.slices)
#pragma unroll
        for (int i = 0; i < 8; i += 2 * step) {
          t[i] = warp_merged(t[i], t[i + step]);
          if (i / (2 * step) % 2) t[i] = __shfl_sync(0xffffffffu, t[i], 31 - lane);
        }
    top = t[0];
  }
  __syncwarp();  // before the lists of the next beam
  if (lane >= K || top == 0) return 0ull;
  const float x = key_logit(top), s = x == -INFINITY ? -INFINITY : base + (x - lse);
  sh.token[beam][lane] = key_token(top);
  return key_of(s != s ? -INFINITY : s, beam * 32 + lane);
}

// Grid (slices, beams, batch). Finished beams have no logits to read: their
// CTAs leave, and the join waits for the others (the first CTA joins where
// all are finished).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) select_kernel(const __grid_constant__ BeamArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams, group = blockIdx.z;
  pdl_launch_dependents();
  pdl_wait();
  uint32_t open;
  if (slice_of_row<T>(a, sh, group, blockIdx.y, blockIdx.x, open)) {
    __syncthreads();
    if (tid == 0) {  // releases this CTA's list and acquires the others'
      sh.last = add_acq_rel(a.arrivals + group, 1) == __popc(open) * a.slices - 1;
      if (sh.last) a.arrivals[group] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
  } else if (open != 0 || blockIdx.x + blockIdx.y != 0) {
    return;
  }
  // Keys order by score, beam and rank: ties go to the lowest beam.
  unsigned long long best = 0;
  for (int beam = warp; beam < K; beam += kWarps) {
    const unsigned long long k = offers_of_row(a, sh, group, beam);
    best = beam == warp ? k : warp_merged(best, __shfl_sync(0xffffffffu, k, 31 - lane));
  }
  for (int half = kWarps / 2; half; half >>= 1) {
    if (K <= half) continue;
    if (warp >= half && warp < 2 * half) sh.kept[warp * 32 + lane] = best;
    __syncthreads();
    if (warp < half) best = warp_merged(best, sh.kept[(warp + half) * 32 + 31 - lane]);
  }
  if (warp != 0) return;
  __syncwarp();
  if (lane < K) {  // every beam has an offer
    const int beam = key_token(best) >> 5 & (kMaxBeams - 1), token = sh.token[beam][key_token(best) & 31];
    const size_t to = (size_t)group * K + lane;
    const bool over = a.finished[group * K + beam] != 0 || token == a.eos;
    a.scores_out[to] = key_logit(best);
    a.parents[to] = beam;
    a.tokens[to] = token;
    a.finished_out[to] = over;
  }
}

// Slices of a row: enough CTAs for about three on every SM, no slice below one
// tile of a CTA, and lists that fit the join.
int slices_of(int rows, int beams, int vocab, int sms) {
  const int most = std::min({beams <= 8 ? 32 : 8, kListKeys / beams, (vocab + kThreads * kElems - 1) / (kThreads * kElems)});
  return std::max(1, std::min(most, (3 * sms + rows - 1) / rows));
}

// (The outputs of an element are written while other CTAs, of finished beams or
// other elements, may still have the inputs to read.)
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

}  // namespace
}  // namespace paged
}  // namespace ce

using namespace ce;
using namespace ce::paged;

extern "C" {

int ce_beam_workspace(int batch, int beams, int vocab, size_t *bytes) {
  CE_REQUIRE(batch >= 1 && batch <= kMaxGroups && beams >= 1 && beams <= kMaxBeams && vocab >= 1,
             "batch must be in [1, %d], beams in [1, %d], vocab >= 1 (got %d, %d, %d)", kMaxGroups, kMaxBeams, batch,
             beams, vocab);
  CE_REQUIRE(bytes != nullptr, "null argument");
  const size_t lists = (size_t)batch * beams * slices_of(1, beams, vocab, 1 << 20);
  *bytes = 4ull * kMaxGroups + lists * 8 * (beams + 1);
  return CE_OK;
}

int ce_beam_select(float *scores_out, int32_t *parents, int32_t *tokens, uint8_t *finished_out, const void *logits,
                   int type, int64_t ld, const float *scores, const uint8_t *finished, int batch, int beams, int vocab,
                   int eos, int pad, void *workspace, size_t workspace_bytes, ce_stream_t stream) {
  size_t need = 0;
  const int rc = ce_beam_workspace(batch, beams, vocab, &need);
  if (rc != CE_OK) return rc;
  CE_REQUIRE(scores_out != nullptr && parents != nullptr && tokens != nullptr && finished_out != nullptr &&
                 logits != nullptr && scores != nullptr && finished != nullptr, "null argument");
  CE_REQUIRE(type == CE_TYPE_F32 || type16(type), "logits must be F32, BF16 or F16 (got %d)", type);
  CE_REQUIRE(reinterpret_cast<uintptr_t>(logits) % type_bytes(type) == 0, "the logits must be aligned to their type");
  CE_REQUIRE(ld >= vocab, "the row stride %lld is shorter than the vocabulary %d", (long long)ld, vocab);
  CE_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
             "the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  const size_t n = (size_t)batch * beams, row = (size_t)type_bytes(type) * vocab;
  const std::pair<const void *, size_t> outputs[] = {{scores_out, 4 * n}, {parents, 4 * n}, {tokens, 4 * n}, {finished_out, n}};
  const std::pair<const void *, size_t> inputs[] = {
      {scores, 4 * n}, {finished, n}, {logits, (n - 1) * (size_t)type_bytes(type) * ld + row}};
  for (const auto &o : outputs)
    for (const auto &i : inputs)
      CE_REQUIRE(!overlap(o.first, o.second, i.first, i.second), "an output lies over an input");
  const int slices = slices_of(batch * beams, beams, vocab, sm_count());
  const size_t lists = (size_t)batch * beams * slices;
  BeamArgs a = {scores_out, parents, tokens, finished_out, logits, ld, scores, finished, batch, beams, vocab, eos, pad,
                slices, static_cast<int *>(workspace), nullptr, nullptr};
  a.best = reinterpret_cast<unsigned long long *>(a.arrivals + kMaxGroups);
  a.sums = reinterpret_cast<float2 *>(a.best + lists * beams);
  const dim3 grid((unsigned)slices, (unsigned)beams, (unsigned)batch);
  auto go = [&](auto kernel) {
    return launch_kernel(kernel, grid, dim3(kThreads), 0, (cudaStream_t)stream, true, "select_kernel", a);
  };
  return type == CE_TYPE_F32 ? go(select_kernel<float>) : type == CE_TYPE_F16 ? go(select_kernel<__half>)
                                                                             : go(select_kernel<__nv_bfloat16>);
}

}  // extern "C"
