// Attention of one new token per request over a paged key-value cache.
//
// For a request and a kv head the G query heads that share it attend to the
// same keys: S^T = K Q^T, O^T = V^T P^T, a matrix product with the keys (or
// the head's dimensions) as the 16-row side and the query heads as the 8-wide
// side. Every key and value is used once, G x 4 flops per element pair, so
// the bound is the memory that K and V come from. The design serves that:
//
//   * The unit of work is 16 or 32 keys of one (request, kv head). All units of
//     the batch form one line, in which every CTA (one per SM), and in it every
//     warp, takes an equal contiguous share, whatever the lengths: a long
//     request is split over many SMs, many short ones share a warp. The change
//     from one request to the next costs a warp about a unit's time, so each
//     has a slot of its own on the line (64 requests of up to 1,024 tokens,
//     one of them a single token: 149 us without that slot, 133 with it).
//     Lengths are read on the device; the grid never depends on them.
//   * A warp runs alone: no block barrier until its share is done. TMA brings
//     its units into a ring of its own, across request boundaries (one 4-D
//     box per 128 bytes of head row and page: head-major and token-major pages
//     are the same to it, and what lies past head_dim or the pool reads as
//     zeros), with an mbarrier per stage. One unit ahead, 64 KB under way on
//     an SM, is best: with two the same batch takes 132 us in the place of
//     127, six documents of up to 100,003 tokens 314 in the place of 294.
//     (Copies by the lanes themselves, 16 bytes each, take 18 instructions a
//     key and 176 us.)
//   * Lanes read shared memory in 16-byte pieces without bank conflicts and
//     without transposing: 16 bytes of a key serve as the lane's part of the
//     contracted dimension (any order will do, when q is laid out alike), and
//     16 bytes of four values are paired by byte permutes into the rows of
//     V^T. Which key takes which row of the product is free too; row g takes
//     key g if even, (g + 4) mod 8 if odd, so that with the 128-byte swizzle
//     the eight lanes of a phase meet eight different bank groups in both.
//   * mma.sync (m16n8k16), not tcgen05: with 8 query heads on the narrow side
//     little is spent on padding, accumulators stay in registers beside the
//     softmax, and the tensor pipe is active 14% of the time (bf16, one query
//     head per kv head; E4M3 with five of them 21%). A tcgen05 tile would have
//     128 rows of queries to fill from at most 16.
//   * The softmax keeps a running reference and sum per query head in fp32.
//     The weights e^(s - reference) enter the second product as two 16-bit
//     parts (the rounded value and what the rounding lost): rounded once to 16
//     bits they would err as much as the output's own rounding. Two bf16 parts
//     hold 16 bits of any weight. Two f16 parts hold 22 of a large one but end
//     at 2^-24, so for f16 and E4M3 caches the reference follows the units'
//     largest scores down as well as up (see the softmax below): it costs
//     nothing where memory is the bound, up to 2% of the other calls (64
//     requests of 1,024 tokens, 32 heads of 128, E4M3: 73.6 and 74.9 us).
//   * A request split over warps or CTAs is joined from (reference, sum, O) parts:
//     within a CTA from shared memory, across CTAs by the last to arrive or,
//     where parts are many, by a launch of their own; in the order of the
//     keys, so the result does not depend on who is last.
//
// Measured (B200, measured copy rate 6.45 TB/s): 64 requests of 32 heads of
// 128, 782 MB of bf16 keys and values, 128 us = 6.1 TB/s; six documents with
// 8 kv heads of 128, 1.99 GB, 297 us = 6.7 TB/s; 96 requests over an E4M3
// cache with 3 kv heads of 96, 123 MB, 37.2 us = 3.3 TB/s, where the bound is
// the chain of instructions per unit (two conversions per four cached bytes,
// a third of the issue slots used by 10 warps); one request of 512 tokens, 12
// heads of 64: 8.9 us, of which the lengths and pages take 2, the unit 1.5,
// the joins 4.
#include <algorithm>
#include <type_traits>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "paged.cuh"

namespace ce {
namespace paged {
namespace {

__device__ DeviceStatus g_attention_status;  // bad pages and lengths
__device__ DeviceStatus g_attention_wait;    // a wait that gave up (it ends the waits of others, too)

// Keys of a unit: 16 where a row of a head takes more than 128 bytes, else 32,
// so that a unit is 8 KB of keys and values at the common head sizes.
constexpr int unit_of(int dim, int item) { return dim > 64 && item == 2 ? 16 : 32; }
constexpr int kMinShare = 4;           // slots of a CTA at least
constexpr int kMaxSplitHeads = 16;     // query heads of one pass over the keys
constexpr int kMaxGrid = 1024;         // CTAs the workspace's counters are laid out for
constexpr int kRowsPerLane = 8;        // requests per lane up to which a warp scans the lengths by itself
constexpr int kPartFloats = kMaxSplitHeads * (128 + 2);

// The request part that a CTA shares with others, for the join across CTAs.
struct Crossing {
  int row, kh, tile, c0, c1;  // and the first and last of its CTAs
};

struct AttnArgs {
  const void *q;
  void *out;
  float *lse;
  const float *k_scale, *v_scale;
  const int32_t *table, *lens;
  long long q_ld, out_ld;
  int seqs, max_pages, pages, heads, kv_heads, dim, shift;
  int group, tiles;  // query heads per kv head; passes over them
  float scale;
  int *arrivals;  // [kMaxGrid], zero between calls
  Crossing *crossings;  // [grid], of the requests that begin in a CTA and end in another; null: joined here
  float *parts;   // [grid][2][kPartFloats]
};

// How many warps a CTA has (by the registers of a warp, 160 to 255 a lane, and
// the shared memory of its ring and parts) and how many units each keeps in
// its ring.
template <int D, int NT, bool F8>
struct Shape {
  static constexpr int kItem = F8 ? 1 : 2;                    // bytes of a cached element
  static constexpr int kKeyChunks = D * kItem / 64;           // 16-byte pieces of a key row per lane
  static constexpr int kValBytes = D * kItem / 8 >= 16 ? 16 : 8;
  static constexpr int kValChunks = D * kItem / 8 / kValBytes;  // pieces of a value row per lane
  static constexpr int kTiles = D * kItem > 128 ? 2 : 1;        // 128-byte wide tiles of kUnit rows
  static constexpr int kUnit = unit_of(D, kItem);
  static constexpr int kHalves = kUnit / 16;                    // products of 16 keys
  static constexpr int kTileBytes = 128 * kUnit;
  static constexpr int kStageBytes = 2 * kTiles * kTileBytes;   // keys, then values
  static constexpr int kWarps = NT == 1 ? (kTiles == 2 ? 8 : D == 128 ? 10 : 12)
                                        : (kTiles == 2 ? 6 : D == 128 ? 8 : 10);
  static constexpr int kStages = 2;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPart = kHeads * (D + 2);  // floats of one (O, max, sum) part
  static constexpr int kVals = D / 8;             // dimensions of a value row per lane
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr size_t kSmem = (size_t)kWarps * (kRing + 4 * kPart);
  static_assert(4 * kPart <= kRing, "a warp's second part lies in its ring");
  static_assert(4 * kThreads <= kWarps * 4 * kPart, "the prefix sums lie in the parts' place");
  static_assert(kSmem <= 230 * 1024, "shared memory of an SM, with 2 KB besides");
};

// One part of a split request as a warp or CTA holds it.
struct Span {
  uint32_t slot;           // the place of its first unit on the line
  int row, kh, tile;       // request, kv head, pass over its query heads
  int k0, k1, units;       // its units of the request's `units`
};

// A box of one page's rows of one head into shared memory (128-byte swizzle).
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int token,
                                              int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(token), "r"(head), "r"(page)
      : "memory");
}

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Four E4M3 values as two f16 pairs (every E4M3 value is an f16 value).
__device__ __forceinline__ void e4m3_to_f16(uint32_t x, uint32_t &lo, uint32_t &hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(x));
}

// (lo, hi) as two 16-bit values of the product's type, and what that lost.
template <bool BF>
__device__ __forceinline__ void split16(float lo, float hi, uint32_t &big, uint32_t &rest) {
  if constexpr (BF) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo - __low2float(b), hi - __high2float(b));
    big = *reinterpret_cast<const uint32_t *>(&b), rest = *reinterpret_cast<const uint32_t *>(&r);
  } else {
    const __half2 b = __floats2half2_rn(lo, hi);
    const __half2 r = __floats2half2_rn(lo - __low2float(b), hi - __high2float(b));
    big = *reinterpret_cast<const uint32_t *>(&b), rest = *reinterpret_cast<const uint32_t *>(&r);
  }
}

template <typename Io>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 b = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&b);
}

__device__ __forceinline__ int row_len(const AttnArgs &a, int b) {
  const long long top = (long long)a.max_pages << a.shift;
  const int len = __ldg(a.lens + b);
  if (len < 0 || len > top) {
    report_timeout(&g_attention_status, kSiteLen);
    return len < 0 ? 0 : (int)top;
  }
  return len;
}

// (unsigned: lengths go up to 2^31 - 1)
template <int UNIT>
__device__ __forceinline__ int units_of(int len) { return (int)(((unsigned)len + UNIT - 1) / UNIT); }
template <int UNIT>
__device__ __forceinline__ int slots_of(int len) { return len > 0 ? units_of<UNIT>(len) + 1 : 0; }

// A place on the line of units. Requests of length 0 have none.
template <int UNIT>
struct Cursor {
  int row, kh, tile, k, len, units;  // request, kv head, pass over its query heads, unit; the request's length and units
  __device__ __forceinline__ void next_row(const AttnArgs &a) {
    do {
      if (++row >= a.seqs) {  // only if the lengths changed under the call: stay inside the buffers
        row = a.seqs - 1, len = 0, units = 1;
        return;
      }
      len = row_len(a, row);
    } while (len == 0);
    units = units_of<UNIT>(len);
  }
  __device__ __forceinline__ void step(const AttnArgs &a) {
    if (++k < units) return;
    k = 0;
    if (++tile < a.tiles) return;
    tile = 0;
    if (++kh < a.kv_heads) return;
    kh = 0;
    next_row(a);
  }
};

// Writes dimensions d .. of query head `head` of a request.
template <typename Io>
__device__ __forceinline__ void store_out8(const AttnArgs &a, int row, int head, int d, const float (&x)[8]) {
  uint4 w;
  w.x = pack2<Io>(x[0], x[1]), w.y = pack2<Io>(x[2], x[3]), w.z = pack2<Io>(x[4], x[5]), w.w = pack2<Io>(x[6], x[7]);
  *reinterpret_cast<uint4 *>(static_cast<Io *>(a.out) + row * a.out_ld + (long long)head * a.dim + d) = w;
}

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

template <typename Io>
__device__ __forceinline__ void store_out4(const AttnArgs &a, int row, int head, int d, float4 x, float f) {
  uint2 w;
  w.x = pack2<Io>(x.x * f, x.y * f), w.y = pack2<Io>(x.z * f, x.w * f);
  *reinterpret_cast<uint2 *>(static_cast<Io *>(a.out) + row * a.out_ld + (long long)head * a.dim + d) = w;
}

__device__ __forceinline__ void add_scaled(float4 &x, float f, float4 y) {
  x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
}

template <int D, int NT, bool F8, typename Io>
__global__ void __launch_bounds__(Shape<D, NT, F8>::kThreads, 1)
attention_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D, NT, F8>;
  constexpr bool BF = !F8 && std::is_same<Io, __nv_bfloat16>::value;  // type of the products
  constexpr int W = S::kWarps, ST = S::kStages, kUnit = S::kUnit, H = S::kHalves;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[W][ST];
  // units of the requests up to each thread's last, per kv head and pass; in
  // the place of the warps' first parts until every warp has found its share
  int *const ends = reinterpret_cast<int *>(smem + (size_t)W * S::kRing);
  __shared__ Span spans[2 * W];
  __shared__ Crossing crossing[2];
  __shared__ int span_used[2 * W], scratch[32], n_crossing, is_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int passes = a.kv_heads * a.tiles;
  pdl_launch_dependents();
  if (tid == 0) {
    n_crossing = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  if (tid < 2 * W) span_used[tid] = 0;
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[warp][i], 1);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  if (a.crossings != nullptr && tid == 0) a.crossings[blockIdx.x].row = -1;

  // ---- the line: for every request, kv head and pass over its query heads a
  // slot for the change to it (fetching q, writing the output: about the time
  // of a unit) and one for each of its units. Prefix sums over the requests, by every warp for
  // itself (no barrier) up to 256 requests, by the CTA together above
  const bool few = a.seqs <= 32 * kRowsPerLane;
  const int per = few ? (a.seqs + 31) / 32 : (a.seqs + S::kThreads - 1) / S::kThreads;
  const int first_row = (few ? lane : tid) * per;
  int lens[kRowsPerLane], mine = 0, sum;
  bool empty = false;
  if (few) {
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) lens[i] = i < per && first_row + i < a.seqs ? row_len(a, first_row + i) : -1;
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) mine += slots_of<kUnit>(lens[i]), empty = empty || lens[i] == 0;
    mine = warp_inclusive_sum(mine);
    sum = __shfl_sync(0xffffffffu, mine, 31);
  } else {
    for (int b = first_row; b < min(a.seqs, first_row + per); ++b) {
      const int len = row_len(a, b);
      mine += slots_of<kUnit>(len);
      empty = empty || len == 0;
    }
    ends[tid] = block_inclusive_sum(mine, scratch, sum);
  }
  if (few ? __any_sync(0xffffffffu, empty) : __syncthreads_or(empty)) {
    const float zero[8] = {};
    for (int b = blockIdx.x + gridDim.x * warp; b < a.seqs; b += gridDim.x * W) {
      if (row_len(a, b) != 0) continue;
      for (int u = lane; u < a.heads * (a.dim >> 3); u += 32)
        store_out8<Io>(a, b, u / (a.dim >> 3), 8 * (u % (a.dim >> 3)), zero);
      for (int h = lane; a.lse != nullptr && h < a.heads; h += 32) a.lse[(size_t)b * a.heads + h] = -INFINITY;
    }
  }
  // Shares of the line: `share` slots a CTA (the last may have less, and
  // CTAs past the line's end none), spread evenly over its warps.
  const uint32_t line = (uint32_t)sum * (uint32_t)passes;
  const uint32_t share = max((line + gridDim.x - 1) / gridDim.x, (uint32_t)kMinShare);
  const uint32_t cta0 = blockIdx.x * share;
  if (cta0 >= line) return;
  const uint32_t cta_slots = min(share, line - cta0);
  uint32_t slot = cta0 + (uint32_t)((uint64_t)cta_slots * warp / W);
  int count = (int)(cta0 + (uint32_t)((uint64_t)cta_slots * (warp + 1) / W) - slot);  // slots left

  const uint32_t ring = smem_u32(smem) + (uint32_t)warp * S::kRing;
  float *const part0 = reinterpret_cast<float *>(smem + (size_t)W * S::kRing) + warp * S::kPart;
  float *const part1 = reinterpret_cast<float *>(smem + (size_t)warp * S::kRing);

  // ---- where the share begins
  Cursor<kUnit> at = {0, 0, 0, 0, 0, 1};
  if (count > 0) {
    uint32_t before;
    if (few) {
      const uint32_t beyond = __ballot_sync(0xffffffffu, (uint64_t)(uint32_t)mine * passes > slot);
      const int lo = beyond ? __ffs(beyond) - 1 : 31;
      int row = first_row, len = 0, sums = mine;
#pragma unroll
      for (int i = 0; i < kRowsPerLane; ++i) sums -= slots_of<kUnit>(lens[i]);  // before this lane's rows
      bool found = false;
#pragma unroll
      for (int i = 0; i < kRowsPerLane; ++i) {
        const int n = slots_of<kUnit>(lens[i]);
        if (!found && n > 0) {
          if ((uint64_t)(uint32_t)(sums + n) * passes > slot) found = true, row = first_row + i, len = lens[i];
          else sums += n;
        }
      }
      at.row = __shfl_sync(0xffffffffu, row, lo), at.len = __shfl_sync(0xffffffffu, len, lo);
      before = __shfl_sync(0xffffffffu, sums, lo);
    } else {
      int lo = 0, hi = S::kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((uint64_t)(uint32_t)ends[mid] * passes > slot) hi = mid; else lo = mid + 1;
      }
      before = lo > 0 ? ends[lo - 1] : 0;
      const int last = min(a.seqs, (lo + 1) * per) - 1;
      for (at.row = lo * per;; ++at.row) {
        at.len = row_len(a, at.row);
        if (at.row >= last || (uint64_t)(before + slots_of<kUnit>(at.len)) * passes > slot) break;
        before += slots_of<kUnit>(at.len);
      }
    }
    at.units = max(1, units_of<kUnit>(at.len));
    const uint32_t in = slot - before * (uint32_t)passes, each = (uint32_t)at.units + 1;
    const int pass = (int)min((uint32_t)passes - 1, in / each);
    at.kh = pass / a.tiles, at.tile = pass % a.tiles;
    at.k = (int)(in - (uint32_t)pass * each) - 1;
    if (at.k < 0) at.k = 0, --count, ++slot;
  }
  if (!few) __syncthreads();  // `ends` gives way to the parts

  if (count > 0) {
    // Copies run ahead of the products by ST - 1 units, page lookups by one
    // more, so that no copy waits for its page id. A unit is one box of a
    // page, or kUnit / page_size boxes of as many pages, one per lane.
    Cursor<kUnit> look = at;  // the unit whose pages are looked up next
    const int32_t *pages = a.table + (size_t)look.row * a.max_pages;
    const int rows = min(kUnit, 1 << a.shift), mask = (1 << a.shift) - 1, sub = lane * rows;  // of this lane's box
    int page = 0, token = 0, head = 0, left = 0;  // of the looked-up unit; left: live keys (less than 1: no unit)
    int to_look = count;
    auto look_up = [&] {
      left = 0;
      if (to_look <= 0) return;
      const unsigned key = (unsigned)look.k * kUnit + sub;
      left = look.len - look.k * kUnit;
      head = look.kh;
      token = (int)(key & mask);
      page = sub < min(left, kUnit) ? __ldg(pages + (key >> a.shift)) : 0;
      to_look -= look.k + 1 == look.units ? 2 : 1;  // the unit's slot, and that of the change to the next request
      if (to_look <= 0) return;
      const int row = look.row;
      look.step(a);
      if (look.row != row) pages = a.table + (size_t)look.row * a.max_pages;
    };
    int to = 0, issued = 0;
    auto issue = [&] {  // copies the looked-up unit into its stage, then looks up the next
      if (left <= 0) return;
      uint64_t *bar = &full[warp][to];
      const int boxes = (min(left, kUnit) + rows - 1) / rows;
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * rows * 128 * 2 * S::kTiles));
      __syncwarp();
      if (lane < boxes) {
        if ((unsigned)page >= (unsigned)a.pages) {
          report_timeout(&g_attention_status, kSitePage);
          page = a.pages;  // past the map: zeros
        }
        const uint32_t dst = ring + (uint32_t)to * S::kStageBytes + (uint32_t)sub * 128;
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
          tma_load_page(dst + i * S::kTileBytes, &k_map, bar, i * (128 / S::kItem), token, head, page);
          tma_load_page(dst + (S::kTiles + i) * S::kTileBytes, &v_map, bar, i * (128 / S::kItem), token, head, page);
        }
      }
      to = to + 1 == ST ? 0 : to + 1;
      ++issued;
      look_up();
    };
    look_up();
#pragma unroll 1
    for (int s = 0; s < ST - 1; ++s) issue();

    // q as it lies in memory, heads 8 nt + g of a pass, dimensions in the order
    // of the keys' pieces. With one tile of heads it is fetched a request part
    // ahead (two tiles leave no registers for that).
    uint4 raw[NT][D / 32];
    auto load_q = [&](const Cursor<kUnit> &c) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = c.tile * S::kHeads + 8 * nt + g;
        const Io *src = static_cast<const Io *>(a.q) + c.row * a.q_ld + (long long)(c.kh * a.group + h) * a.dim;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          // runs of 8: for 16-bit caches piece t + 4i, for 8-bit ones half of a piece of 16
          const int d = F8 ? 16 * (t + 4 * (i >> 1)) + 8 * (i & 1) : 8 * (t + 4 * i);
          raw[nt][i] = h < a.group && d < a.dim ? __ldg(reinterpret_cast<const uint4 *>(src + d)) : make_uint4(0, 0, 0, 0);
        }
      }
    };
    if constexpr (NT == 1) load_q(at);
    const uint8_t *const ring_ptr = smem + (size_t)warp * S::kRing;

    // ---- the share
    uint32_t q[NT][D / 8];       // this lane's part of the contracted dimension, heads 8 nt + g
    float cs[NT][2];             // score factor (base 2) of heads 8 nt + 2t, + 1
    float m[NT][2], l[NT][2];    // running maximum (base 2) and this lane's sum
    float o[NT][S::kVals / 2][4];
    int k0 = at.k;               // first unit of the current request part
    uint32_t start = slot;
    bool fresh = true, first_part = true;
    // Row g of the products stands for key pi, row g + 8 for pi + 8.
    const int pi = g & 1 ? (g + 4) & 7 : g, pe = 2 * t, po = (2 * t + 5) & 7;  // pi of g, 2t, 2t + 1
    uint32_t key_at[2], val_at[2];  // this lane's pieces in a stage
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      key_at[p] = pi * 128 + (((t + 4 * p) ^ pi) << 4);
      const int key = p ? po : pe;
      val_at[p] = S::kTiles * S::kTileBytes + key * 128 +
                  (S::kValBytes == 16 ? (g ^ key) << 4 : (((g >> 1) ^ key) << 4) + 8 * (g & 1));
    }
    int stage = 0, landed = 0;
    uint32_t parity = 0;
    for (;;) {
      if (fresh) {
        fresh = false;
        if constexpr (NT > 1) load_q(at);
        const int kh = at.kh;
        const float ks = a.k_scale != nullptr ? __ldg(a.k_scale + kh) : 1.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f = a.scale * kLog2e * ks;
          if constexpr (F8) {
            // The 8-bit cache's products are f16. q is brought into f16's
            // range by a power of two per head (exact but for elements 2^-14
            // below the largest), which the score factor takes back.
            float x[D / 4], top = 0.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              const Io *e = reinterpret_cast<const Io *>(&raw[nt][c]);
#pragma unroll
              for (int i = 0; i < 8; ++i) x[8 * c + i] = to_float(e[i]), top = fmaxf(top, fabsf(x[8 * c + i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e above top, kept where both powers are normal
            const int e = min(126, max(-126, (int)(__float_as_uint(top) >> 23) - 126));
            const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) q[nt][i] = pack2<__half>(x[2 * i] * down, x[2 * i + 1] * down);
            f *= up;
          } else {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
              q[nt][4 * c] = raw[nt][c].x, q[nt][4 * c + 1] = raw[nt][c].y, q[nt][4 * c + 2] = raw[nt][c].z,
              q[nt][4 * c + 3] = raw[nt][c].w;
          }
          // the factor of head 8 nt + g lives in lanes 4g ..; this lane's columns are 2t, 2t + 1
          cs[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
          cs[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
          m[nt][0] = m[nt][1] = -INFINITY;
          l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
          for (int i = 0; i < S::kVals / 2; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        if (NT == 1 && count - (at.units - at.k) > 1) {
          Cursor<kUnit> next = at;
          next.k = next.units - 1;
          next.step(a);
          load_q(next);
        }
      }
      if (!warp_wait(&full[warp][stage], parity, &g_attention_wait, kSiteWait)) break;
      ++landed;
      issue();  // into the stage that the previous unit left
      const uint8_t *const st = ring_ptr + (uint32_t)stage * S::kStageBytes;
      const bool tail = at.k + 1 == at.units;     // may have keys past the length
      const int n_live = at.len - at.k * kUnit;
      // The values of the first 16 keys are on their way from shared memory
      // during the scores.
      constexpr int kWords = S::kValBytes * S::kValChunks / 4;
      uint32_t x[4][kWords];
      auto load_values = [&](int hf) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < S::kValChunks; ++c) {
            const uint8_t *from = st + val_at[r & 1] + c * S::kTileBytes + (2 * hf + (r >> 1)) * (8 * 128);
            if constexpr (S::kValBytes == 16) {
              const uint4 y = *reinterpret_cast<const uint4 *>(from);
              x[r][4 * c] = y.x, x[r][4 * c + 1] = y.y, x[r][4 * c + 2] = y.z, x[r][4 * c + 3] = y.w;
            } else {
              const uint2 y = *reinterpret_cast<const uint2 *>(from);
              x[r][0] = y.x, x[r][1] = y.y;
            }
          }
        if (tail) {  // weights of 0 must meet values of 0, whatever the cache holds there
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((r & 1 ? po : pe) + 8 * (r >> 1) + 16 * hf >= n_live)
#pragma unroll
              for (int w = 0; w < kWords; ++w) x[r][w] = 0;
        }
      };
      // ---- scores: 16 keys x 8 NT heads per half, in sums of their own so that no product waits long
      constexpr int kSums = 2 * S::kKeyChunks * H > 4 ? 4 / H : 2;
      float s[NT][H][4];
#pragma unroll
      for (int hf = 0; hf < H; ++hf) {
        uint4 kx[S::kKeyChunks][2];
#pragma unroll
        for (int c = 0; c < S::kKeyChunks; ++c)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            kx[c][r] = *reinterpret_cast<const uint4 *>(st + key_at[c & 1] + (c >> 1) * S::kTileBytes +
                                                        (2 * hf + r) * (8 * 128));
        if (hf == 0) load_values(0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sums[kSums][4];
#pragma unroll
          for (int y = 0; y < kSums; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[y][i] = 0.f;
#pragma unroll
          for (int c = 0; c < S::kKeyChunks; ++c) {
            const uint32_t xw[4] = {kx[c][0].x, kx[c][0].y, kx[c][0].z, kx[c][0].w};
            const uint32_t yw[4] = {kx[c][1].x, kx[c][1].y, kx[c][1].z, kx[c][1].w};
            if constexpr (F8) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t x0, x1, y0, y1;
                e4m3_to_f16(xw[j], x0, x1);
                e4m3_to_f16(yw[j], y0, y1);
                mma<BF>(sums[(4 * c + j) % kSums], x0, y0, x1, y1, q[nt][8 * c + 2 * j], q[nt][8 * c + 2 * j + 1]);
              }
            } else {
              mma<BF>(sums[2 * c % kSums], xw[0], yw[0], xw[1], yw[1], q[nt][4 * c], q[nt][4 * c + 1]);
              mma<BF>(sums[(2 * c + 1) % kSums], xw[2], yw[2], xw[3], yw[3], q[nt][4 * c + 2], q[nt][4 * c + 3]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y = sums[0][i] + sums[1][i];
            if constexpr (kSums == 4) y += sums[2][i] + sums[3][i];
            s[nt][hf][i] = y * cs[nt][i & 1];
          }
        }
      }
      // ---- softmax: keys of rows g (elements 0, 1) and g + 8 (2, 3), heads 2t, 2t + 1.
      // The weights are 2^(s - m) of a reference m near the unit's largest
      // score. It moves only when that score leaves a window about it, so that
      // most units need a vote instead of a reduction and a rescaling. For
      // bf16 parts, with fp32's exponents, the window has an upper end alone.
      // f16 parts end at 2^-24: weights far below the largest so far (an
      // attention sink, say) would keep few bits or none. So m follows the
      // scores down, and a unit's largest weight is between 2^-9 and 2^15.9,
      // 2^11 where m has been set: what a weight loses below 2^-25 is at most
      // 2^-16 of the unit's largest. O and l, in fp32, thereby grow to
      // 2^kRoom at most; from there on m stays.
      if (tail) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int hf = 0; hf < H; ++hf)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pi + 8 * (i >> 1) + 16 * hf >= n_live) s[nt][hf][i] = -INFINITY;
      }
      constexpr float kBelow = BF ? 0.f : 11.f;  // m is set this far below the unit's largest score
      constexpr float kUp = BF ? 8.f : 15.875f, kDown = -9.f;
      constexpr int kRoom = 64;
      auto largest = [&](int nt, int j) {
        float top = fmaxf(s[nt][0][j], s[nt][0][j + 2]);
        if constexpr (H == 2) top = fmaxf(top, fmaxf(s[nt][1][j], s[nt][1][j + 2]));
        return top;
      };
      bool moved = false;
      if constexpr (BF) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) moved = moved || largest(nt, j) > m[nt][j] + kUp;
        moved = __any_sync(0xffffffffu, moved);
      } else {
        uint32_t seen = 0;  // a bit per head with a score not too low, and one for a score too high
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float above = largest(nt, j) - m[nt][j];
            if (above >= kDown) seen |= 1u << (2 * nt + j);
            if (above > kUp) seen |= 0x80000000u >> (2 * NT * t);
          }
        seen = __reduce_or_sync(0xffffffffu, seen << (2 * NT * t));
        moved = seen != (1u << (8 * NT)) - 1u;
      }
      if (moved) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = largest(nt, j);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
            float mn = fmaxf(m[nt][j], top - kBelow);
            if constexpr (!BF) {
              float most = l[nt][j];
#pragma unroll
              for (int y = 4; y < 32; y <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, y));
              const int room = kRoom + 126 - (int)(__float_as_uint(most) >> 23);  // most < 2^(kRoom - room)
              if (top > -INFINITY && top - m[nt][j] < kDown)
                mn = fmaxf(top - kBelow, m[nt][j] - (float)min(max(room, 0), kRoom));
            }
            const float f = mn == -INFINITY ? 1.f : exp2_approx(m[nt][j] - mn);
            m[nt][j] = mn;
            l[nt][j] *= f;
#pragma unroll
            for (int i = 0; i < S::kVals / 2; ++i) o[nt][i][j] *= f, o[nt][i][j + 2] *= f;
          }
      }
      uint32_t big[NT][H][2], rest[NT][H][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) base[j] = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
#pragma unroll
        for (int hf = 0; hf < H; ++hf) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = exp2_approx(s[nt][hf][i] - base[i & 1]);
          l[nt][0] += p[0] + p[2];
          l[nt][1] += p[1] + p[3];
          split16<BF>(p[0], p[1], big[nt][hf][0], rest[nt][hf][0]);
          split16<BF>(p[2], p[3], big[nt][hf][1], rest[nt][hf][1]);
#pragma unroll
          for (int r = 0; r < 2; ++r)
            big[nt][hf][r] = transpose8x8(big[nt][hf][r]), rest[nt][hf][r] = transpose8x8(rest[nt][hf][r]);
        }
      }
      // ---- values: rows of V^T are this lane's kVals dimensions, in pairs (i, i + kVals / 2)
#pragma unroll
      for (int hf = 0; hf < H; ++hf) {
        if (hf > 0) load_values(hf);
        constexpr int kPer = 4 / S::kItem;  // elements of a word
#pragma unroll
        for (int i = 0; i < S::kVals / 2; i += 2) {
          uint32_t v[2][4];  // elements i and i + 1: (row g | g + 8) x (keys 2t, 2t + 1 | 2t + 8, 2t + 9)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int e = i + (r & 1) * (S::kVals / 2), w = e / kPer, pr = 2 * (r >> 1);
            if constexpr (F8) {
              e4m3_to_f16(__byte_perm(x[pr][w], x[pr + 1][w], e % kPer ? 0x7362 : 0x5140), v[0][r], v[1][r]);
            } else {
              v[0][r] = __byte_perm(x[pr][w], x[pr + 1][w], 0x5410);
              v[1][r] = __byte_perm(x[pr][w], x[pr + 1][w], 0x7632);
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma<BF>(o[nt][i + u], v[u][0], v[u][1], v[u][2], v[u][3], big[nt][hf][0], big[nt][hf][1]);
              mma<BF>(o[nt][i + u], v[u][0], v[u][1], v[u][2], v[u][3], rest[nt][hf][0], rest[nt][hf][1]);
            }
        }
      }
      if (++stage == ST) stage = 0, parity ^= 1u;

      // ---- end of the request's keys, or of the share
      const bool ends_here = at.k + 1 == at.units;
      --count, ++slot;
      const bool over = count == 0 || (ends_here && count == 1);
      if (ends_here || over) {
        const int kh = at.kh, h0 = at.tile * S::kHeads;
        const bool whole = ends_here && k0 == 0;
        const float vs = a.v_scale != nullptr ? __ldg(a.v_scale + kh) : 1.f;
        const int place = first_part ? 0 : 1;
        float *part = place ? part1 : part0;
        if (place && !whole) __syncwarp();  // the ring is the second part's place: every lane is done with the last unit
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float sum = l[nt][j];
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
            const int h = 8 * nt + 2 * t + j;
            const bool live = h0 + h < a.group;
            const float f = whole ? vs / sum : 1.f;
            constexpr int kRun = S::kValBytes / S::kItem;  // consecutive dimensions of a piece
#pragma unroll
            for (int e0 = 0; e0 < S::kVals; e0 += 8) {
              const int d = (g + 8 * (e0 / kRun)) * kRun + e0 % kRun;
              float y[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int e = e0 + i;
                y[i] = o[nt][e % (S::kVals / 2)][j + 2 * (e / (S::kVals / 2))] * f;
              }
              if (!live) continue;
              if (!whole) {
                *reinterpret_cast<float4 *>(part + h * D + d) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(part + h * D + d + 4) = make_float4(y[4], y[5], y[6], y[7]);
              } else if (d < a.dim) {
                store_out8<Io>(a, at.row, kh * a.group + h0 + h, d, y);
              }
            }
            if (g == 0 && live) {
              if (!whole) {
                part[S::kHeads * D + 2 * h] = m[nt][j];
                part[S::kHeads * D + 2 * h + 1] = sum;
              } else if (a.lse != nullptr) {
                a.lse[(size_t)at.row * a.heads + kh * a.group + h0 + h] = m[nt][j] * kLn2 + logf(sum);
              }
            }
          }
        if (!whole && lane == 0) {
          spans[2 * warp + place] = {start, at.row, at.kh, at.tile, k0, at.k + 1, at.units};
          span_used[2 * warp + place] = 1;
        }
        if (over) break;
        fresh = true, first_part = false;
        --count;
        start = ++slot;
        k0 = 0;
      }
      at.step(a);
    }
    // After a wait that gave up: no copy may land in the memory of a CTA that has left.
    for (; landed < issued; ++landed) {
      warp_wait(&full[warp][stage], parity, nullptr, kSiteWait);
      if (++stage == ST) stage = 0, parity ^= 1u;
    }
  }
  __syncthreads();

  // ---- parts of the CTA's warps, joined in the order of the keys. Lane e
  // looks at part e; a run of parts of one request begins where the request
  // changes, and the runs go round the warps.
  auto warp_part = [&](int e) {
    const int w = e >> 1;
    return (e & 1) ? reinterpret_cast<const float *>(smem + (size_t)w * S::kRing)
                   : reinterpret_cast<const float *>(smem + (size_t)W * S::kRing) + w * S::kPart;
  };
  {
    const bool used = lane < 2 * W && span_used[lane];
    const Span mine = used ? spans[lane] : Span{0, -1, 0, 0, 0, 0, 0};
    const uint32_t parts = __ballot_sync(0xffffffffu, used);
    const uint32_t below = parts & ((1u << lane) - 1u);
    const int prev = below ? 31 - __clz(below) : 0;
    // (every lane takes part in every shuffle: no short-circuit around them)
    const int prev_row = __shfl_sync(0xffffffffu, mine.row, prev), prev_kh = __shfl_sync(0xffffffffu, mine.kh, prev);
    const int prev_tile = __shfl_sync(0xffffffffu, mine.tile, prev);
    const bool other = prev_row != mine.row || prev_kh != mine.kh || prev_tile != mine.tile;
    const uint32_t begins = __ballot_sync(0xffffffffu, used && (below == 0 || other));
    // 4 dimensions of a head of a run per thread
    const int widest = min(S::kHeads, a.group), tasks = widest * (D / 4), all = __popc(begins) * tasks;
    for (int u = tid; u < all; u += S::kThreads) {
      uint32_t rest = begins;
      for (int r = u / tasks; r > 0; --r) rest &= rest - 1;
      const int e0 = __ffs(rest) - 1, h = u % tasks / (D / 4), d = 4 * (u % (D / 4)), ml = S::kHeads * D + 2 * h;
      rest &= rest - 1;
      const uint32_t members = parts & ~((1u << e0) - 1u) & (rest ? (rest & -rest) - 1u : ~0u);
      const Span &first = spans[e0];
      const int h0 = first.tile * S::kHeads, head = first.kh * a.group + h0 + h;
      if (h0 + h >= a.group) continue;
      float m = -INFINITY;
      for (uint32_t b = members; b; b &= b - 1) m = fmaxf(m, warp_part(__ffs(b) - 1)[ml]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t b = members; b; b &= b - 1) {
        const float *p = warp_part(__ffs(b) - 1);
        const float f = exp2_approx(p[ml] - base);
        l += f * p[ml + 1];
        add_scaled(x, f, *reinterpret_cast<const float4 *>(p + h * D + d));
      }
      if (first.k0 == 0 && spans[31 - __clz(members)].k1 == first.units) {
        const float vs = a.v_scale != nullptr ? __ldg(a.v_scale + first.kh) : 1.f;
        if (d < a.dim) store_out4<Io>(a, first.row, head, d, x, vs / l);
        if (d == 0 && a.lse != nullptr) a.lse[(size_t)first.row * a.heads + head] = m * kLn2 + logf(l);
      } else {
        // across CTAs: place 1 holds the part of a request that begins in this
        // CTA, place 0 of one that began before
        float *const place = a.parts + ((size_t)blockIdx.x * 2 + (first.k0 == 0)) * kPartFloats;
        __stcg(reinterpret_cast<float4 *>(place + h * D + d), x);
        if (d == 0) {
          __stcg(reinterpret_cast<float2 *>(place + ml), make_float2(m, l));
          if (h == 0) {  // CTAs of the request's first and last unit
            const uint32_t b0 = first.slot - first.k0;
            crossing[atomicAdd(&n_crossing, 1)] = {first.row, first.kh, first.tile, (int)(b0 / share),
                                                   (int)((b0 + first.units - 1) / share)};
          }
        }
      }
    }
  }
  __syncthreads();
  if (n_crossing == 0) return;
  if (a.crossings != nullptr) {  // join_kernel does the rest
    if (tid < n_crossing && crossing[tid].c0 == (int)blockIdx.x) a.crossings[blockIdx.x] = crossing[tid];
    return;
  }
  if (tid < n_crossing) {
    // releases the CTA's part (written before the barrier) and acquires the others'
    const Crossing c = crossing[tid];
    is_last[tid] = add_acq_rel(a.arrivals + c.c0, 1) == c.c1 - c.c0;
    if (is_last[tid]) a.arrivals[c.c0] = 0;
  }
  __syncthreads();
  // ---- the last CTA of a request joins the CTAs' parts: weights of the parts
  // per head by a warp each, then 4 dimensions per thread, the parts shared
  // out over the threads that are left
  for (int x = 0; x < n_crossing; ++x) {
    if (!is_last[x]) continue;
    const Crossing c = crossing[x];
    const int n = c.c1 - c.c0 + 1, h0 = c.tile * S::kHeads, heads = min(S::kHeads, a.group - h0);
    const int head0 = c.kh * a.group + h0, tasks = heads * (D / 4);
    const float vs = a.v_scale != nullptr ? __ldg(a.v_scale + c.kh) : 1.f;
    auto part = [&](int i) { return a.parts + ((size_t)(c.c0 + i) * 2 + (i == 0)) * kPartFloats; };
    float4 *const sums = reinterpret_cast<float4 *>(smem);                     // [groups][tasks]
    float *const inv = reinterpret_cast<float *>(sums + S::kThreads);          // [heads] v_scale / sum
    float2 *const weight = reinterpret_cast<float2 *>(inv + S::kHeads);        // [heads][n]
    for (int u = tid; u < heads * n; u += S::kThreads)
      weight[u] = __ldcg(reinterpret_cast<const float2 *>(part(u % n) + S::kHeads * D + 2 * (u / n)));
    __syncthreads();
    for (int h = warp; h < heads; h += W) {
      float m = -INFINITY;
      for (int i = lane; i < n; i += 32) m = fmaxf(m, weight[h * n + i].x);
#pragma unroll
      for (int y = 16; y; y >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < n; i += 32) {
        const float f = exp2_approx(weight[h * n + i].x - base);
        l += f * weight[h * n + i].y;
        weight[h * n + i].x = f;
      }
#pragma unroll
      for (int y = 16; y; y >>= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
      if (lane == 0) {
        inv[h] = vs / l;
        if (a.lse != nullptr) a.lse[(size_t)c.row * a.heads + head0 + h] = m * kLn2 + logf(l);
      }
    }
    __syncthreads();
    // kOwn tasks of a thread side by side, so that enough reads are under way
    constexpr int kOwn = (S::kHeads * D / 4 + S::kThreads - 1) / S::kThreads;
    const int groups = max(1, S::kThreads / tasks), group = groups > 1 ? tid / tasks : 0;
    const int task0 = groups > 1 ? tid % tasks : tid;
    float4 y[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; ++o) y[o] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (group < groups) {
      // (reads past the last part or task are of the last one, with weight 0)
      for (int i0 = group; i0 < n; i0 += 4 * groups) {
        float4 x[4][kOwn];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float4 *const from = reinterpret_cast<const float4 *>(part(min(i0 + u * groups, n - 1)));
#pragma unroll
          for (int o = 0; o < kOwn; ++o) x[u][o] = __ldcg(from + min(task0 + o * S::kThreads, tasks - 1));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int o = 0; o < kOwn; ++o) {
            const int i = i0 + u * groups, task = task0 + o * S::kThreads;
            const float w = weight[min(task, tasks - 1) / (D / 4) * n + min(i, n - 1)].x;
            add_scaled(y[o], i < n ? w : 0.f, x[u][o]);
          }
      }
    }
    if (groups > 1) {
      if (group < groups) sums[tid] = y[0];
      __syncthreads();
      if (tid < tasks)
        for (int i = 1; i < groups; ++i) add_scaled(y[0], 1.f, sums[i * tasks + tid]);
    }
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      const int task = tid + o * S::kThreads, h = task / (D / 4), d = 4 * (task % (D / 4));
      if (task < tasks && d < a.dim) store_out4<Io>(a, c.row, head0 + h, d, y[o], inv[h]);
    }
    __syncthreads();
  }
}

// The join across CTAs as a launch of its own: block (c, h) joins the parts of
// query head h of the request that begins in CTA c and ends in a later one.
constexpr int kJoinThreads = 256;
template <int D, int HEADS, typename Io>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float2 weight[kMaxGrid];
  __shared__ float4 sums[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 31, h = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  const Crossing c = a.crossings[blockIdx.x];
  if (c.row < 0 || h >= a.group - c.tile * HEADS) return;
  const int n = c.c1 - c.c0 + 1, head = c.kh * a.group + c.tile * HEADS + h;
  auto part = [&](int i) { return a.parts + ((size_t)(c.c0 + i) * 2 + (i == 0)) * kPartFloats; };
  for (int i = tid; i < n; i += kJoinThreads)
    weight[i] = __ldcg(reinterpret_cast<const float2 *>(part(i) + HEADS * D + 2 * h));
  __syncthreads();
  float m = -INFINITY, l = 0.f;  // by every warp for itself
  for (int i = lane; i < n; i += 32) m = fmaxf(m, weight[i].x);
#pragma unroll
  for (int y = 16; y; y >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
  const float base = m == -INFINITY ? 0.f : m;
  for (int i = lane; i < n; i += 32) l += exp2_approx(weight[i].x - base) * weight[i].y;
#pragma unroll
  for (int y = 16; y; y >>= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
  constexpr int kGroups = kJoinThreads / (D / 4);
  const int d = 4 * (tid % (D / 4)), group = tid / (D / 4);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = group; i0 < n; i0 += 4 * kGroups) {
    float4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x[u] = __ldcg(reinterpret_cast<const float4 *>(part(min(i0 + u * kGroups, n - 1)) + h * D + d));
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kGroups;
      add_scaled(sum, i < n ? exp2_approx(weight[min(i, n - 1)].x - base) : 0.f, x[u]);
    }
  }
  sums[tid] = sum;
  __syncthreads();
  if (group > 0) return;
  for (int i = 1; i < kGroups; ++i) add_scaled(sum, 1.f, sums[i * (D / 4) + tid]);
  const float vs = a.v_scale != nullptr ? __ldg(a.v_scale + c.kh) : 1.f;
  if (d < a.dim) store_out4<Io>(a, c.row, head, d, sum, vs / l);
  if (tid == 0 && a.lse != nullptr) a.lse[(size_t)c.row * a.heads + head] = m * kLn2 + logf(l);
}

template <int D, int NT, bool F8, typename Io>
int launch_attention(const AttnArgs &a, const CUtensorMap (&maps)[2], int grid, cudaStream_t s) {
  using S = Shape<D, NT, F8>;
  static bool done[64] = {};
  int dev = 0;
  CE_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !done[dev]) {
    CE_CUDA_TRY(cudaFuncSetAttribute(attention_kernel<D, NT, F8, Io>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)S::kSmem));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  const int rc = launch_kernel(attention_kernel<D, NT, F8, Io>, dim3((unsigned)grid), dim3(S::kThreads), S::kSmem, s,
                               true, "attention_kernel", a, maps[0], maps[1]);
  if (rc != CE_OK || a.crossings == nullptr) return rc;
  return launch_kernel(join_kernel<D, S::kHeads, Io>, dim3((unsigned)grid, (unsigned)std::min(S::kHeads, a.group)),
                       dim3(kJoinThreads), 0, s, true, "join_kernel", a);
}

template <bool F8, typename Io>
int dispatch_attention(const AttnArgs &a, const CUtensorMap (&maps)[2], int grid, cudaStream_t s) {
  if (a.dim <= 64)
    return a.group <= 8 ? launch_attention<64, 1, F8, Io>(a, maps, grid, s) : launch_attention<64, 2, F8, Io>(a, maps, grid, s);
  return a.group <= 8 ? launch_attention<128, 1, F8, Io>(a, maps, grid, s) : launch_attention<128, 2, F8, Io>(a, maps, grid, s);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p) : nullptr;
  }();
  return fn;
}

// The map of one layer of a pool: [pages][heads][tokens][head_dim] with the
// pool's strides; boxes of 128 bytes x min(unit, page_size) tokens.
int make_page_map(CUtensorMap *map, const ce_paged_kv *kv, void *pool, int layer, int unit_keys) {
  const auto fn = encode_fn();
  if (fn == nullptr) return set_error(CE_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int b = type_bytes(kv->type);
  const cuuint64_t dims[4] = {(cuuint64_t)kv->head_dim, (cuuint64_t)kv->page_size, (cuuint64_t)kv->kv_heads,
                              (cuuint64_t)kv->pages};
  // the stride of a dimension of size 1 is never used; any that the map takes will do
  auto stride = [&](int64_t elements, int size) { return size > 1 ? (cuuint64_t)elements * b : (cuuint64_t)16; };
  const cuuint64_t strides[3] = {stride(kv->token_stride, kv->page_size), stride(kv->head_stride, kv->kv_heads),
                                 stride(kv->page_stride, kv->pages)};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / b), (cuuint32_t)std::min(unit_keys, kv->page_size), 1, 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  char *base = static_cast<char *>(pool) + (long long)layer * kv->layer_stride * b;
  // Fetches widened to 256 bytes suit rows of whole 128-byte pieces, and rows
  // of one head that follow one another; beside others they bring other heads'
  // rows (3 heads of 96 bytes, token-major: 39.7 us with 256, 36.6 with 64; 32
  // heads of 256 bytes: 127.9 and 128.4; 12 heads of 224 bytes, head-major:
  // 112 and 117).
  const bool apart = kv->head_dim * b % 128 != 0 && kv->token_stride != kv->head_dim;
  const CUtensorMapL2promotion fetch = apart ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  const CUresult r = fn(map, b == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims,
                        strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        fetch, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CE_OK : set_error(CE_ERR_CUDA, format("cuTensorMapEncodeTiled failed (%d)", (int)r));
}

size_t workspace_bytes_of(int grid) {
  return 4ull * kMaxGrid + (size_t)grid * (2 * kPartFloats * 4 + sizeof(Crossing));
}

// Whether the joins across CTAs are a launch of their own. One CTA reads the
// parts of a request at about 40 bytes a cycle; where few requests share the
// whole grid these are many. (Lengths are on the device, so the rule goes by
// the mean: a long request among many short ones has more parts than it
// expects and is still joined by the last CTA.) 30,000 tokens, 2 kv heads of 128, one request:
// 16 query heads each (600 KB of parts a kv head) 41.5 us joined by the last
// CTA, 20.6 with the launch; 4 heads (150 KB) 17.0 and 14.7; four requests
// of 4,000 tokens, 2 kv heads of 96, 8 query heads each (55 KB) 15.8 and
// 11.2. Below that the launch's 2 us of host time weigh more than the 0.5 to
// 1 us of the device's that it saves (one request, 12 heads of 64, 3 KB: 8.7
// and 8.2 us on the device, 6.8 and 9 on the host).
bool join_apart(const AttnArgs &a, int grid) {
  const long long items = (long long)a.seqs * a.kv_heads * a.tiles;
  const long long bytes = grid / items * std::min(a.group, kMaxSplitHeads) * a.dim * 4;  // of a request's parts, at most
  return bytes > 32 * 1024;
}

}  // namespace
}  // namespace paged

using namespace paged;

// Reads and clears the status words of the attention kernels.
int paged_attention_status() {
  CE_CUDA_TRY(cudaDeviceSynchronize());
  DeviceStatus bad{}, wait{};
  CE_CUDA_TRY(cudaMemcpyFromSymbol(&bad, g_attention_status, sizeof(bad)));
  CE_CUDA_TRY(cudaMemcpyFromSymbol(&wait, g_attention_wait, sizeof(wait)));
  if (bad.code == 0 && wait.code == 0) return CE_OK;
  const DeviceStatus zero{};
  CE_CUDA_TRY(cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero)));
  CE_CUDA_TRY(cudaMemcpyToSymbol(g_attention_wait, &zero, sizeof(zero)));
  if (wait.code != 0)
    return set_error(CE_ERR_TIMEOUT, format("paged attention: a copy did not land in time (block %u)", wait.block));
  return set_error(CE_ERR_USAGE, bad.where == kSitePage ? "paged attention: a page id lies outside the pool"
                                                        : "paged attention: a length does not fit its table row");
}

int paged_attention_set_wait_limit(unsigned long long ns) { return set_wait_limit_here(ns); }

}  // namespace ce

using namespace ce;

extern "C" {

int ce_paged_attention_workspace(size_t *bytes) {
  CE_REQUIRE(bytes != nullptr, "null argument");
  *bytes = workspace_bytes_of(std::min(sm_count(), kMaxGrid));
  return CE_OK;
}

int ce_paged_attention(const ce_paged_kv *kv, int layer, const ce_page_table *pt, void *out, float *lse,
                       const void *q, int io_type, int heads, int64_t q_ld, int64_t out_ld, float scale,
                       void *workspace, size_t workspace_bytes, ce_stream_t stream) {
  int rc = check_kv(kv, layer);
  if (rc == CE_OK) rc = check_table(pt, "pages");
  if (rc != CE_OK) return rc;
  CE_REQUIRE(kv->pages == pt->pages && kv->page_size == pt->page_size,
             "the cache has %d pages of %d, the block table %d of %d", kv->pages, kv->page_size, pt->pages,
             pt->page_size);
  CE_REQUIRE(q != nullptr && out != nullptr, "null q or out");
  CE_REQUIRE(type16(io_type) && (kv->type == CE_TYPE_E4M3 || io_type == kv->type),
             "q and out must be of the cache's type, or BF16 or F16 for an E4M3 cache (got %d, cache %d)", io_type,
             kv->type);
  CE_REQUIRE(heads >= 1 && heads % kv->kv_heads == 0, "heads must be a multiple of kv_heads (got %d, %d)", heads,
             kv->kv_heads);
  const int64_t row = (int64_t)heads * kv->head_dim;
  CE_REQUIRE(aligned16(q) && aligned16(out) && q_ld % 8 == 0 && out_ld % 8 == 0 && q_ld >= row && out_ld >= row,
             "q and out must be 16-byte aligned, their row strides multiples of 8 and at least heads * head_dim");
  const int grid = std::min(sm_count(), kMaxGrid);
  const size_t need = workspace_bytes_of(grid);
  CE_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
             "the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  AttnArgs a = {};
  CUtensorMap maps[2];
  const int unit = unit_of(kv->head_dim, type_bytes(kv->type));
  rc = make_page_map(&maps[0], kv, kv->k_dev, layer, unit);
  if (rc == CE_OK) rc = make_page_map(&maps[1], kv, kv->v_dev, layer, unit);
  if (rc != CE_OK) return rc;
  a.q = q, a.out = out, a.lse = lse;
  a.k_scale = kv->k_scale_dev, a.v_scale = kv->v_scale_dev;
  a.table = pt->table_dev, a.lens = pt->lens_dev;
  a.q_ld = q_ld, a.out_ld = out_ld;
  a.seqs = pt->seqs, a.max_pages = pt->max_pages, a.pages = kv->pages;
  a.heads = heads, a.kv_heads = kv->kv_heads, a.dim = kv->head_dim, a.shift = log2_of(kv->page_size);
  a.group = heads / kv->kv_heads;
  a.tiles = a.group <= 8 ? 1 : (a.group + kMaxSplitHeads - 1) / kMaxSplitHeads;
  a.scale = scale;
  const int64_t slots = (int64_t)pt->max_pages * pt->page_size / unit + 2;  // slots of a full row at most
  CE_REQUIRE(pt->seqs * slots < (1ll << 31) && (double)pt->seqs * slots * kv->kv_heads * a.tiles < 4294967296.0 - kMaxGrid,
             "seqs x max_pages x page_size x kv_heads is too large (%d x %d x %d x %d)", pt->seqs, pt->max_pages,
             pt->page_size, kv->kv_heads);
  a.arrivals = static_cast<int *>(workspace);
  a.parts = reinterpret_cast<float *>(a.arrivals + kMaxGrid);
  a.crossings = join_apart(a, grid) ? reinterpret_cast<Crossing *>(a.parts + (size_t)grid * 2 * kPartFloats) : nullptr;
  const cudaStream_t s = (cudaStream_t)stream;
  if (kv->type == CE_TYPE_BF16) return dispatch_attention<false, __nv_bfloat16>(a, maps, grid, s);
  if (kv->type == CE_TYPE_F16) return dispatch_attention<false, __half>(a, maps, grid, s);
  return io_type == CE_TYPE_F16 ? dispatch_attention<true, __half>(a, maps, grid, s)
                                : dispatch_attention<true, __nv_bfloat16>(a, maps, grid, s);
}

}  // extern "C"
