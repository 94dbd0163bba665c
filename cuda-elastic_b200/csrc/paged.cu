// Block tables and cache writes of the paged key-value cache: resize
// (request lengths -> pages, slots, positions), append (rotary positions and
// the cache write) and reorder (rows follow their beam search parents).
//
// Page allocation needs no free list: a page is free when no row holds it
// (refs 0), and the i-th page that a call takes is the i-th lowest free one.
// So the answer depends on the inputs alone, never on the order in which
// threads arrive: counts of references are sums of integers, and ranks among
// free pages and among rows are prefix sums.
//
// Measured (B200): resize of 64 requests by a token each over 4,096 pages 7.3
// us, of 1,021 requests with 60 prompts (61,000 tokens) over 98,304 pages 23
// us; both are chains of dependent reads, barriers and code run once, far
// from any rate. Reorder of 4 beams, 12 layers 8.3 us, of 128 beams, 32 layers
// 15 us. Append of 8,190 tokens of 32 + 2 x 8 heads of 128, bf16 into an
// E4M3 cache, 34 us = 5.5 TB/s; of 64 tokens of 32 + 2 x 32 heads, fp32 into
// bf16, 2.1 us.
#include <algorithm>

#include "paged.cuh"

namespace ce {
namespace paged {
namespace {

__device__ DeviceStatus g_paged_status;

constexpr int kTableThreads = 1024;
constexpr int kMaxCapacity = 0x7fffffff - 127;  // new tokens of a resize, numbered by ints a warp's 128 at a time

// ---------------------------------------------------------------------------
// Pieces that resize and reorder share

struct Tables {
  const int32_t *table_in, *lens_in, *refs_in;
  int32_t *table, *lens, *refs;
  int32_t *status;
  int n, max_pages, pages, shift;  // rows, columns, pool, log2(page_size)
};

__device__ __forceinline__ int pages_of(int len, int shift) {
  return (int)(((long long)len + (1 << shift) - 1) >> shift);
}

// A length as the tables can hold it (a caller's mistake is cut, not followed).
__device__ __forceinline__ int held_len(const Tables &t, int i) {
  const long long top = (long long)t.max_pages << t.shift;
  const int len = t.lens_in[i];
  if (len < 0 || len > top) {
    report_timeout(&g_paged_status, kSiteLen);
    return len < 0 ? 0 : (int)(top < 0x7fffffff ? top : 0x7fffffff);
  }
  return len;
}

__device__ __forceinline__ bool page_ok(const Tables &t, int page) {
  if ((unsigned)page < (unsigned)t.pages) return true;
  report_timeout(&g_paged_status, kSitePage);
  return false;
}

// The CTA's place in its cluster.
struct Cluster {
  int rank, ranks;
};
__device__ __forceinline__ Cluster this_cluster() {
  int n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return {(int)cluster_ctarank(), n};
}
__device__ __forceinline__ void sync_all(Cluster c) {
  if (c.ranks == 1) __syncthreads(); else cluster_sync();
}

__device__ __forceinline__ int clamp_int(long long v) { return v > 0x7fffffffll ? 0x7fffffff : (int)v; }

// The map of free pages, one bit each, in shares: CTA r of the cluster keeps
// the words of pages [r per, (r + 1) per), per a multiple of 32.
struct FreeMap {
  uint32_t *words;  // this CTA's
  int *ends;        // prefix sums of their free pages, after count()
  int per, lo, hi;
  __device__ __forceinline__ FreeMap(uint32_t *w, int pages, Cluster c) : words(w) {
    per = ((pages + c.ranks - 1) / c.ranks + 31) / 32 * 32;
    lo = min(pages, c.rank * per);
    hi = min(pages, lo + per);
    ends = reinterpret_cast<int *>(w + per / 32);
  }
  // Reads refs once: the map, and the copy into `t.refs` where that is another buffer.
  __device__ __forceinline__ void fill(const Tables &t) const {
    const int lane = threadIdx.x & 31;
    for (int p0 = lo + (int)threadIdx.x - lane; p0 < hi; p0 += blockDim.x * 4) {
      int v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + i * (int)blockDim.x + lane;
        v[i] = p < hi ? __ldcg(t.refs_in + p) : 1;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + i * (int)blockDim.x + lane;
        const uint32_t word = __ballot_sync(0xffffffffu, v[i] == 0);
        if (p < hi && t.refs != t.refs_in) t.refs[p] = v[i];
        if (lane == 0 && p < hi) words[(p - lo) >> 5] = word;
      }
    }
  }
  // A page that has lost its last holder.
  __device__ __forceinline__ void set(int page) const {
    const int r = page / per, in = page - r * per;
    const uint32_t word = cluster_map(smem_u32(words + (in >> 5)), (uint32_t)r);
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(word), "r"(1u << (in & 31)) : "memory");
  }
  // Prefix sums over the words; the number of free pages of the share.
  __device__ __forceinline__ int count(int *scratch) const {
    const int n = (hi - lo + 31) >> 5;
    int base = 0;
    for (int w0 = 0; w0 < n; w0 += blockDim.x) {
      const int w = w0 + threadIdx.x;
      int total;
      const int sum = block_inclusive_sum(w < n ? __popc(words[w]) : 0, scratch, total);
      if (w < n) ends[w] = base + sum;
      base += total;
    }
    return base;
  }
  // The r-th free page of the share (r from 0, below count()).
  __device__ __forceinline__ int nth(int r) const {
    const int w = first_above(ends, (hi - lo + 31) >> 5, r);
    uint32_t bits = words[w];
    r -= w ? ends[w - 1] : 0;
    int at = 0;
#pragma unroll
    for (int half = 16; half; half >>= 1) {  // the half word that holds the r-th set bit
      const int n = __popc(bits & ((1u << half) - 1u));
      if (r >= n) r -= n, bits >>= half, at += half;
    }
    return lo + 32 * w + at;
  }
};

// By one warp, four entries of a lane at a time so that their latencies overlap:
// the pages of a row change their count of holders, or a row is copied.
__device__ __forceinline__ void change_refs(const Tables &t, const FreeMap &map, const int32_t *row, int n, int delta) {
  for (int j = threadIdx.x & 31; j < n; j += 128) {
    int page[4], now[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) page[u] = j + 32 * u < n ? row[j + 32 * u] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool live = j + 32 * u < n && page_ok(t, page[u]);
      now[u] = live ? atomicAdd(t.refs + page[u], delta) + delta : 1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (now[u] == 0) map.set(page[u]);
  }
}
__device__ __forceinline__ void copy_row(int32_t *to, const int32_t *from, int n) {
  for (int j = threadIdx.x & 31; j < n; j += 128) {
    int page[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) page[u] = j + 32 * u < n ? from[j + 32 * u] : 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j + 32 * u < n) to[j + 32 * u] = page[u];
  }
}

// Free pages of the CTAs before this one, and of all.
__device__ __forceinline__ void free_before(int *count, Cluster c, int &before, int &total) {
  before = total = 0;
  const uint32_t here = smem_u32(count);
  for (int r = 0; r < c.ranks; ++r) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_map(here, (uint32_t)r)) : "memory");
    before += r < c.rank ? v : 0;
    total += v;
  }
}

// Inclusive sums over the block of two values per thread.
struct Pair {
  long long a, b;
};
__device__ __forceinline__ Pair block_inclusive_sums(Pair v, Pair *scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v.a = warp_inclusive_sum(v.a), v.b = warp_inclusive_sum(v.b);
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  Pair e = lane < warps ? scratch[lane] : Pair{0, 0};
  e.a = warp_inclusive_sum(e.a), e.b = warp_inclusive_sum(e.b);
  const long long a = __shfl_sync(0xffffffffu, e.a, max(0, warp - 1)), b = __shfl_sync(0xffffffffu, e.b, max(0, warp - 1));
  return {v.a + (warp > 0 ? a : 0), v.b + (warp > 0 ? b : 0)};
}

// ---------------------------------------------------------------------------
// resize

struct ResizeArgs {
  Tables t;
  const int32_t *new_lens;
  int64_t *slots;
  int32_t *pos, *starts;
  int capacity;
};

// One cluster; its time is a chain of dependent reads and barriers, so each
// input is read once, early, and phases that have nothing to do are skipped.
// Every CTA goes over all rows (they are few, and sums over them are needed
// everywhere) and over its share of the pages:
//   1. lengths into shared memory, the free map (and copy) of refs;
//   2. if a row gets shorter: its pages lose a holder (integer atomics), the
//      last holder's loss sets the page's bit in the map;
//   3. each row's need of pages and tokens, and their prefix sums;
//   4. page r of those needed is the r-th free one: the rank is looked up in
//      the map's prefix sums, its row and column in the rows';
//   5. slots and positions, token by token, by the rows' prefix sums.
__global__ void __launch_bounds__(kTableThreads) resize_kernel(const __grid_constant__ ResizeArgs a) {
  extern __shared__ int smem[];
  __shared__ Pair scratch16[32];
  __shared__ int scratch4[32];
  __shared__ int s_free, s_pages, s_tokens, s_refused;
  const Tables &t = a.t;
  const int n = t.n, tid = threadIdx.x, lane = tid & 31, mask = (1 << t.shift) - 1;
  const Cluster c = this_cluster();
  int *need_end = smem, *tok_end = smem + n, *old_len = smem + 2 * n, *new_len = smem + 3 * n;
  const FreeMap map(reinterpret_cast<uint32_t *>(smem + 4 * n), t.pages, c);
  pdl_launch_dependents();
  if (tid == 0) s_pages = s_tokens = s_refused = 0;
  pdl_wait();

  // 1.
  bool shorter = false;
  for (int i = tid; i < n; i += blockDim.x) {
    const int len = a.new_lens[i], old = held_len(t, i);
    old_len[i] = old;
    new_len[i] = len < 0 ? old : len;
    shorter = shorter || (len >= 0 && len < old) || t.table != t.table_in;
  }
  map.fill(t);
  shorter = __syncthreads_or(shorter);
  // 2. (with another table: the rows that stay, too)
  if (shorter) {
    sync_all(c);  // every CTA's share of refs is copied
    const int warps = c.ranks * (int)(blockDim.x >> 5);
    for (int i = c.rank * (int)(blockDim.x >> 5) + (tid >> 5); i < n; i += warps) {
      const int have = pages_of(old_len[i], t.shift), want = pages_of(new_len[i], t.shift);
      const int32_t *row = t.table_in + (size_t)i * t.max_pages;
      change_refs(t, map, row + want, have - want, -1);
      if (t.table != t.table_in) copy_row(t.table + (size_t)i * t.max_pages, row, min(want, have));
    }
  }
  sync_all(c);
  // 3.
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int r0 = min(n, tid * per), r1 = min(n, r0 + per);
  long long need_sum = 0, tok_sum = 0;
  int growing = 0, granted = 0;
  for (int i = r0; i < r1; ++i) {
    const int old = old_len[i], len = new_len[i];
    const int have = pages_of(old, t.shift), want = pages_of(len, t.shift);
    bool fits = len > old && want <= t.max_pages;
    growing += len > old;
    if (fits && (old & mask) != 0) {  // its last page is partly filled
      const int tail = t.table_in[(size_t)i * t.max_pages + (old >> t.shift)];
      fits = page_ok(t, tail) && __ldcg(t.refs + tail) == 1;
    }
    need_sum += fits ? want - have : 0;
    tok_sum += fits ? len - old : 0;
    need_end[i] = clamp_int(need_sum);  // made absolute below
    tok_end[i] = fits ? clamp_int(tok_sum) : -1 - clamp_int(tok_sum);  // sign: does not fit
  }
  const int free = map.count(scratch4);
  if (tid == 0) s_free = free;
  const Pair ends = block_inclusive_sums(Pair{need_sum, tok_sum}, scratch16);
  const long long need0 = ends.a - need_sum, tok0 = ends.b - tok_sum;
  sync_all(c);
  int before, total_free;
  free_before(&s_free, c, before, total_free);
  int pages_given = 0, tokens_given = 0;
  for (int i = r0; i < r1; ++i) {
    const bool fits = tok_end[i] >= 0;
    const int need = clamp_int(need0 + need_end[i]), tok = clamp_int(tok0 + (fits ? tok_end[i] : -1 - tok_end[i]));
    need_end[i] = need, tok_end[i] = tok;
    if (fits && need <= total_free && tok <= a.capacity) pages_given = need, tokens_given = tok, ++granted;
  }
  if (granted) atomicMax(&s_pages, pages_given), atomicMax(&s_tokens, tokens_given);
  if (growing != granted) atomicAdd(&s_refused, growing - granted);
  __syncthreads();
  const int R = s_pages, T = s_tokens;
  // 4.
  for (int r = before + tid; r < min(R, before + free); r += blockDim.x) {
    const int page = map.nth(r - before), i = first_above(need_end, n, r);
    const int col = pages_of(old_len[i], t.shift) + r - (i ? need_end[i - 1] : 0);
    t.table[(size_t)i * t.max_pages + col] = page;
    t.refs[page] = 1;
  }
  sync_all(c);
  // 5. (no CTA reads the old lengths any more)
  const int threads = c.ranks * (int)blockDim.x, first = c.rank * (int)blockDim.x + tid;
  // A warp takes 32 tokens, or 128 where there are more tokens than threads:
  // mostly those of one request, whose row it then looks up once.
  const int runs = a.capacity <= threads ? 1 : 4;
  for (long long b = (long long)(first >> 5) * 32 * runs; b < a.capacity; b += (long long)threads * runs) {
    const int base = (int)b, row = base < T ? first_above(tok_end, n, base) : 0;
    const bool one = base < T && tok_end[row] >= min(T, base + 32 * runs);
    int pos[4], page[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = base + 32 * u + lane;
      pos[u] = -1, page[u] = 0;
      if (u < runs && j < T) {
        const int i = one ? row : first_above(tok_end, n, j);
        pos[u] = old_len[i] + j - (i ? tok_end[i - 1] : 0);
        page[u] = __ldcg(t.table + (size_t)i * t.max_pages + (pos[u] >> t.shift));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = base + 32 * u + lane;
      if (u < runs && j < a.capacity) {
        a.slots[j] = pos[u] < 0 ? -1ll : ((long long)page[u] << t.shift) + (pos[u] & mask);
        a.pos[j] = pos[u];
      }
    }
  }
  for (int i = first; i < n; i += threads) {
    const int start = i ? tok_end[i - 1] : 0, old = old_len[i], len = new_len[i];
    const bool given = tok_end[i] > start && tok_end[i] <= T && need_end[i] <= R;
    t.lens[i] = given || len < old ? len : old;
    if (a.starts != nullptr) a.starts[i] = min(start, T);
  }
  if (c.rank == 0 && tid == 0) {
    if (a.starts != nullptr) a.starts[n] = T;
    if (t.status != nullptr) {
      t.status[0] = R;
      t.status[1] = s_refused;
      t.status[2] = total_free - R;
      t.status[3] = T;
    }
  }
}

// ---------------------------------------------------------------------------
// reorder

struct ReorderArgs {
  Tables t;
  const int32_t *parents;
  int beams;
  int32_t *copies;
};

// One cluster, in the manner of resize_kernel:
//   1. each new row's parent, length and partly filled last page, the
//      children of each old row, the free map;
//   2. refs of every page of old row i change by (children of i) - 1, and
//      each new row's pages are those of its parent. A page comes to 0 only
//      when every row that held it is without children, so whoever brings it
//      there may set its bit, whatever the order;
//   3. rows whose last page another row holds too need a page of their own,
//      all but the first of the group when the group alone holds it;
//   4. the free pages of the lowest ranks go to those rows.
__global__ void __launch_bounds__(kTableThreads) reorder_kernel(const __grid_constant__ ReorderArgs a) {
  extern __shared__ int smem[];
  __shared__ int scratch4[32];
  __shared__ int s_free;
  const Tables &t = a.t;
  const int n = t.n, K = a.beams, tid = threadIdx.x, mask = (1 << t.shift) - 1;
  const Cluster c = this_cluster();
  int *new_len = smem, *tail = smem + n, *copy_end = smem + 2 * n, *children = smem + 3 * n;
  const FreeMap map(reinterpret_cast<uint32_t *>(smem + 4 * n), t.pages, c);
  pdl_launch_dependents();
  for (int i = tid; i < n; i += blockDim.x) children[i] = 0;
  __syncthreads();
  pdl_wait();

  // 1.
  for (int i = tid; i < n; i += blockDim.x) {
    const int p = a.parents[i], src = i - i % K + p;
    const bool kept = p >= 0 && p < K;
    const int len = kept ? held_len(t, src) : 0;
    int page = -1;
    if ((len & mask) != 0) {
      page = t.table_in[(size_t)src * t.max_pages + (len >> t.shift)];
      if (!page_ok(t, page)) page = -1;
    }
    if (kept) atomicAdd(children + src, 1);
    new_len[i] = len;
    tail[i] = page;
  }
  map.fill(t);
  sync_all(c);
  // 2.
  const int warps = c.ranks * (int)(blockDim.x >> 5);
  for (int i = c.rank * (int)(blockDim.x >> 5) + (tid >> 5); i < n; i += warps) {
    const int held = pages_of(new_len[i], t.shift), delta = children[i] - 1;
    const int32_t *from = t.table_in + (size_t)(i - i % K + (held ? a.parents[i] : 0)) * t.max_pages;
    const int32_t *mine = t.table_in + (size_t)i * t.max_pages;
    const int have = delta != 0 ? pages_of(held_len(t, i), t.shift) : 0;
    copy_row(t.table + (size_t)i * t.max_pages, from, held);
    change_refs(t, map, mine, have, delta);
  }
  sync_all(c);
  // 3.
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int r0 = min(n, tid * per), r1 = min(n, r0 + per);
  int want = 0;
  for (int i = r0; i < r1; ++i) {
    const int page = tail[i], g = i - i % K;
    if (page >= 0) {
      const int refs = __ldcg(t.refs + page);
      int holders = 0, first = K;
      for (int k = K - 1; k >= 0; --k)
        if (tail[g + k] == page) ++holders, first = k;
      want += !(first == i - g && refs == holders);
    }
    copy_end[i] = want;  // made absolute below
  }
  const int free = map.count(scratch4);
  if (tid == 0) s_free = free;
  int wanted;
  const int want0 = block_inclusive_sum(want, scratch4, wanted) - want;
  for (int i = r0; i < r1; ++i) copy_end[i] += want0;
  sync_all(c);
  int before, total_free;
  free_before(&s_free, c, before, total_free);
  const int R = min(wanted, total_free);
  // 4.
  for (int r = before + tid; r < min(R, before + free); r += blockDim.x) {
    const int page = map.nth(r - before), i = first_above(copy_end, n, r);
    t.table[(size_t)i * t.max_pages + (new_len[i] >> t.shift)] = page;
    t.refs[page] = 1;
    atomicAdd(t.refs + tail[i], -1);
    a.copies[2 * i] = tail[i];
    a.copies[2 * i + 1] = page;
  }
  const int threads = c.ranks * (int)blockDim.x;
  for (int i = c.rank * (int)blockDim.x + tid; i < n; i += threads) {
    const int r = i ? copy_end[i - 1] : 0;
    if (copy_end[i] == r || r >= R) a.copies[2 * i] = a.copies[2 * i + 1] = -1;
    t.lens[i] = new_len[i];
  }
  if (c.rank == 0 && tid == 0 && t.status != nullptr) {
    t.status[0] = R;
    t.status[1] = wanted - R;
    t.status[2] = total_free - R;
    t.status[3] = R;
  }
  if (c.ranks > 1) cluster_sync();  // no CTA leaves while another reads its free count
}

// The page copies of a reorder: 16-byte pieces of the len % page_size tokens
// of every copied row, in all layers, K and V: read and written once. Each
// CTA lists the rows that copy (the host does not know them), then takes
// (row, layer) pairs in turn; blockIdx.y shares out the pieces of a pair
// where pairs alone would not fill the GPU.
struct CopyArgs {
  const int32_t *copies, *lens;
  char *k, *v;
  long long layer_stride, page_stride, head_stride, token_stride;  // bytes
  int rows, layers, kv_heads, pieces, page_size;                   // pieces: 16-byte pieces of a head's row
};
constexpr int kCopyThreads = 256;

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  __shared__ unsigned short list[kMaxRows];
  __shared__ int scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  int listed = 0;
  uint32_t few = 0;  // up to 32 rows a warp lists by itself, in a word
  if (a.rows <= 32) {
    const int lane = threadIdx.x & 31;
    few = __ballot_sync(0xffffffffu, lane < a.rows && a.copies[2 * lane] >= 0);
    listed = __popc(few);
  }
  for (int r0 = 0; a.rows > 32 && r0 < a.rows; r0 += kCopyThreads) {
    const int r = r0 + threadIdx.x;
    const int copied = r < a.rows && a.copies[2 * r] >= 0;
    int total;
    const int at = listed + block_inclusive_sum(copied, scratch, total) - 1;
    if (copied) list[at] = (unsigned short)r;
    listed += total;
  }
  if (a.rows > 32) __syncthreads();
  const int step = gridDim.y * kCopyThreads;
  for (long long p = blockIdx.x; p < (long long)listed * a.layers; p += gridDim.x) {
    const int at_row = (int)(p / a.layers), layer = (int)(p % a.layers);
    int row;
    if (a.rows <= 32) {
      uint32_t rest = few;
      for (int i = 0; i < at_row; ++i) rest &= rest - 1;
      row = __ffs(rest) - 1;
    } else {
      row = list[at_row];
    }
    const int src = a.copies[2 * row], dst = a.copies[2 * row + 1], tokens = a.lens[row] & (a.page_size - 1);
    const int total = tokens * a.kv_heads * a.pieces;
    char *const k = a.k + layer * a.layer_stride, *const v = a.v + layer * a.layer_stride;
    for (int u0 = blockIdx.y * kCopyThreads + threadIdx.x; u0 < total; u0 += 2 * step) {
      uint4 x[2], y[2];
      long long at[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned u = min(u0 + i * step, total - 1), rest = u / (unsigned)a.pieces;
        at[i] = (rest / (unsigned)tokens) * a.head_stride + (rest % (unsigned)tokens) * a.token_stride +
                16ll * (u % (unsigned)a.pieces);
        x[i] = *reinterpret_cast<const uint4 *>(k + at[i] + src * a.page_stride);
        y[i] = *reinterpret_cast<const uint4 *>(v + at[i] + src * a.page_stride);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (u0 + i * step < total) {
          *reinterpret_cast<uint4 *>(k + at[i] + dst * a.page_stride) = x[i];
          *reinterpret_cast<uint4 *>(v + at[i] + dst * a.page_stride) = y[i];
        }
    }
  }
}

// ---------------------------------------------------------------------------
// append

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out;
  char *kc, *vc;  // layer base
  const float *k_scale, *v_scale;
  const int64_t *slots;
  const int32_t *pos;
  const float *rope;
  long long q_ld, k_ld, v_ld;
  long long page_stride, head_stride, token_stride;  // elements
  long long slot_end;                                // pages * page_size
  int tokens, heads, kv_heads, dim, shift, rope_len;
};

// Eight elements as they lie in memory.
template <typename T>
struct Row8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
  }
  __device__ __forceinline__ void widen(float (&x)[8]) const {
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(e[i]);
  }
};

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
  uint4 o;
  __nv_bfloat162 *e = reinterpret_cast<__nv_bfloat162 *>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4 *>(p) = o;
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
  uint4 o;
  __half2 *e = reinterpret_cast<__half2 *>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4 *>(p) = o;
}
__device__ __forceinline__ void store8(__nv_fp8_e4m3 *p, const float (&x)[8]) {
  uint2 o;
  __nv_fp8x2_storage_t *e = reinterpret_cast<__nv_fp8x2_storage_t *>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<uint2 *>(p) = o;
}

// A thread has 8 elements (4 rotary pairs) at one place of up to Heads heads of
// a token (q, k and v heads numbered one after the other), in fp32, rounded
// once where they are stored. Blocks are (head_dim / 8, heads): no index is
// divided and the scales are multiplied by their reciprocals, since the
// threads are short and issue slots count beside the memory (206 instructions
// a thread with the divisions, 159 without). The slot and the position are
// fetched at once, behind the heads: one link less in the chain from the slot
// to the rotary row is 42 -> 40 us at 8,190 tokens of 32 + 2 x 8 heads of 128,
// bf16 into E4M3, and three heads for one look-up 34.6 us. Every element is
// read and written once. Six CTAs of three heads to an SM cost 8 to 20 bytes
// of spills a thread and are worth it: 33.3 us, 34.2 with five and none.
constexpr int kAppendThreads = 256;
template <typename In, typename Out, typename Cache, int Heads>
__global__ void __launch_bounds__(kAppendThreads, Heads == 1 ? 8 : 6) append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_launch_dependents();
  const int all = a.heads + 2 * a.kv_heads, step = gridDim.y * blockDim.y;
  const int first = blockIdx.y * blockDim.y + threadIdx.y;
  if (first >= all) return;
  const int d = 8 * threadIdx.x, tok = blockIdx.x;
  const In *q = static_cast<const In *>(a.q) + tok * a.q_ld + d;
  const In *k = static_cast<const In *>(a.k) + tok * a.k_ld + d;
  const In *v = static_cast<const In *>(a.v) + tok * a.v_ld + d;
  Out *q_out = static_cast<Out *>(a.q_out) + (long long)tok * a.heads * a.dim + d;
  pdl_wait();
  Row8<In> in[Heads];
#pragma unroll
  for (int i = 0; i < Heads; ++i) {  // on their way while the slot and position are looked up
    int h = first + i * step;
    if (h >= all) break;
    const In *src = h < a.heads ? q : h < a.heads + a.kv_heads ? k : v;
    h -= h < a.heads ? 0 : h < a.heads + a.kv_heads ? a.heads : a.heads + a.kv_heads;
    in[i].load(src + h * a.dim);
  }
  const long long slot = a.slots[tok];
  const int pos = a.rope != nullptr ? a.pos[tok] : 0;
  bool live = slot >= 0;
  if (live && slot >= a.slot_end) {
    report_timeout(&g_paged_status, kSiteSlot);
    live = false;
  }
  if (live && a.rope != nullptr && (pos < 0 || pos >= a.rope_len)) {
    report_timeout(&g_paged_status, kSitePos);
    live = false;
  }
  if (!live) {
    const float zero[8] = {};
    for (int h = first; h < a.heads; h += step) store8(q_out + h * a.dim, zero);
    return;
  }
  float4 c[2] = {{1, 0, 1, 0}, {1, 0, 1, 0}};  // (cos, sin) of four pairs
  if (a.rope != nullptr) {
    const float4 *cs = reinterpret_cast<const float4 *>(a.rope + (long long)pos * a.dim + d);
    c[0] = __ldg(cs), c[1] = __ldg(cs + 1);
  }
  const long long at = (slot >> a.shift) * a.page_stride + (slot & ((1ll << a.shift) - 1)) * a.token_stride + d;
#pragma unroll
  for (int i = 0; i < Heads; ++i) {
    int h = first + i * step;
    if (h >= all) break;
    float x[8];
    in[i].widen(x);
    if (h < a.heads + a.kv_heads && a.rope != nullptr) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x0 = x[4 * j], x1 = x[4 * j + 1], x2 = x[4 * j + 2], x3 = x[4 * j + 3];
        x[4 * j] = x0 * c[j].x - x1 * c[j].y, x[4 * j + 1] = x0 * c[j].y + x1 * c[j].x;
        x[4 * j + 2] = x2 * c[j].z - x3 * c[j].w, x[4 * j + 3] = x2 * c[j].w + x3 * c[j].z;
      }
    }
    if (h < a.heads) {
      store8(q_out + h * a.dim, x);
      continue;
    }
    h -= a.heads;
    const bool is_v = h >= a.kv_heads;
    if (is_v) h -= a.kv_heads;
    const float *scale = is_v ? a.v_scale : a.k_scale;
    if (scale != nullptr) {
      const float inv = 1.f / __ldg(scale + h);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= inv;
    }
    store8(reinterpret_cast<Cache *>(is_v ? a.vc : a.kc) + at + h * a.head_stride, x);
  }
}

// Launches one cluster of `ranks` CTAs (a table kernel).
template <typename Args>
int launch_tables(void (*kernel)(Args), const Args &a, int ranks, size_t smem, cudaStream_t s, const char *what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ranks);
  cfg.blockDim = dim3(kTableThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  return e == cudaSuccess ? CE_OK : cuda_error(e, what);
}

// Dynamic shared memory of a table kernel: four words per row, and the free
// map and its sums of a CTA's share of the pages.
size_t table_smem(const ce_page_table *t, int ranks) {
  const int words = ((t->pages + ranks - 1) / ranks + 31) / 32;
  return 16ull * t->seqs + 8ull * words;
}
constexpr size_t kTableSmemMax = 16ull * kMaxRows + kMaxPages / 8 / 4 + 128;  // a cluster of 8
static_assert(kTableSmemMax <= 224 * 1024, "a table kernel's shared memory");

// CTAs of a resize: one, whose barriers are cheap, or a cluster of 16 (the
// non-portable size), which costs about 5,500 cycles more in barriers and
// divides the rest: 0.25 cycles per page and 1.4 per token on one CTA. 64
// requests, 4,096 pages: 6.7 us against 10.0; 1,021 requests, 98,304 pages,
// 61,000 tokens: 83 us against 23.
int resize_ranks(const ce_page_table *t, int capacity) {
  return t->pages + 6ll * capacity > 26000 || t->seqs > kTableThreads ? 16 : 1;
}
// Of a reorder: its rows are a warp's work each, 32 of them at once in a CTA.
// 4 rows: 8.4 us on one CTA, 10.2 on eight; 128 rows of 41 pages: 18.6 and 15.0.
int reorder_ranks(const ce_page_table *t) { return t->seqs > 32 || t->pages > 26000 ? 8 : 1; }

// Opts the table kernels into their shared memory, once per device.
int configure_tables() {
  static bool done[64] = {};
  int dev = 0;
  CE_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && done[dev]) return CE_OK;
  CE_CUDA_TRY(cudaFuncSetAttribute(resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTableSmemMax));
  CE_CUDA_TRY(cudaFuncSetAttribute(reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)kTableSmemMax));
  CE_CUDA_TRY(cudaFuncSetAttribute(resize_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (dev >= 0 && dev < 64) done[dev] = true;
  return CE_OK;
}

int check_pair(const ce_page_table *to, const ce_page_table *from) {
  int rc = check_table(from, "from");
  if (rc == CE_OK) rc = check_table(to, "to");
  if (rc != CE_OK) return rc;
  CE_REQUIRE(to->seqs == from->seqs && to->max_pages == from->max_pages && to->pages == from->pages &&
                 to->page_size == from->page_size,
             "`to` and `from` must have the same rows, columns, pages and page size");
  return CE_OK;
}

Tables tables_of(const ce_page_table *to, const ce_page_table *from, int32_t *status) {
  return {from->table_dev, from->lens_dev, from->refs_dev, to->table_dev, to->lens_dev, to->refs_dev, status,
          from->seqs, from->max_pages, from->pages, log2_of(from->page_size)};
}

// Three heads a thread where 16-bit rows fill more than two waves of CTAs
// three times over (4,096 tokens of 32 + 2 x 32 heads of 128: 40.6 us with one
// head, 36.0 with three; 256 tokens: 3.4 and 3.7). Fp32 rows have as many bytes
// in flight with one (48.2 and 48.9 us), and fewer than three heads to a
// thread leave lanes idle (4,096 tokens of 28 + 2 x 4 heads of 96: 13.2, 14.3).
template <typename In, typename Out, typename Cache>
int launch_append(const AppendArgs &a, dim3 grid, dim3 block, cudaStream_t s) {
  if constexpr (sizeof(In) == 2) {
    const long long wave = (long long)sm_count() * (2048 / kAppendThreads);
    if (grid.y >= 3 && (long long)grid.x * grid.y > 2 * wave) {
      grid.y = (grid.y + 2) / 3;
      return launch_kernel(append_kernel<In, Out, Cache, 3>, grid, block, 0, s, true, "append_kernel", a);
    }
  }
  return launch_kernel(append_kernel<In, Out, Cache, 1>, grid, block, 0, s, true, "append_kernel", a);
}

template <typename In, typename Out>
int launch_append(int cache_type, const AppendArgs &a, dim3 grid, dim3 block, cudaStream_t s) {
  if (cache_type == CE_TYPE_BF16) return launch_append<In, Out, __nv_bfloat16>(a, grid, block, s);
  if (cache_type == CE_TYPE_F16) return launch_append<In, Out, __half>(a, grid, block, s);
  return launch_append<In, Out, __nv_fp8_e4m3>(a, grid, block, s);
}

template <typename In>
int launch_append(int out_type, int cache_type, const AppendArgs &a, dim3 grid, dim3 block, cudaStream_t s) {
  return out_type == CE_TYPE_F16 ? launch_append<In, __half>(cache_type, a, grid, block, s)
                                 : launch_append<In, __nv_bfloat16>(cache_type, a, grid, block, s);
}

}  // namespace

int check_kv(const ce_paged_kv *kv, int layer) {
  CE_REQUIRE(kv != nullptr, "null cache");
  CE_REQUIRE(type16(kv->type) || kv->type == CE_TYPE_E4M3, "cache type must be BF16, F16 or E4M3 (got %d)", kv->type);
  CE_REQUIRE(kv->k_dev != nullptr && kv->v_dev != nullptr, "null k or v pool");
  CE_REQUIRE(kv->type == CE_TYPE_E4M3 || (kv->k_scale_dev == nullptr && kv->v_scale_dev == nullptr),
             "a 16-bit cache takes no scales");
  CE_REQUIRE(kv->layers >= 1 && kv->kv_heads >= 1 && kv->pages >= 1 && kv->pages <= kMaxPages,
             "layers and kv_heads must be >= 1 and pages in [1, %d] (got %d, %d, %d)", kMaxPages, kv->layers,
             kv->kv_heads, kv->pages);
  CE_REQUIRE(kv->page_size >= 1 && kv->page_size <= kMaxPage && (kv->page_size & (kv->page_size - 1)) == 0,
             "page_size must be a power of two in [1, %d] (got %d)", kMaxPage, kv->page_size);
  CE_REQUIRE(kv->head_dim >= 16 && kv->head_dim <= 128 && kv->head_dim % 16 == 0,
             "head_dim must be a multiple of 16 in [16, 128] (got %d)", kv->head_dim);
  CE_REQUIRE(layer >= 0 && layer < kv->layers, "layer %d of %d", layer, kv->layers);
  const int64_t unit = 16 / type_bytes(kv->type);
  CE_REQUIRE(aligned16(kv->k_dev) && aligned16(kv->v_dev) && kv->layer_stride % unit == 0 &&
                 kv->page_stride % unit == 0 && kv->head_stride % unit == 0 && kv->token_stride % unit == 0,
             "the cache's bases and strides must be multiples of 16 bytes");
  auto bad = [](int64_t stride, int size) { return stride < 0 || stride >= (1ll << 36) || (size > 1 && stride == 0); };
  CE_REQUIRE(!bad(kv->layer_stride, kv->layers) && !bad(kv->page_stride, kv->pages) &&
                 !bad(kv->head_stride, kv->kv_heads) && !bad(kv->token_stride, kv->page_size),
             "the cache's strides must be positive and below 2^36 elements");
  return CE_OK;
}

int check_table(const ce_page_table *t, const char *what) {
  CE_REQUIRE(t != nullptr, "null page table (%s)", what);
  CE_REQUIRE(t->table_dev != nullptr && t->lens_dev != nullptr && t->refs_dev != nullptr,
             "null buffer in the page table (%s)", what);
  CE_REQUIRE(t->seqs >= 1 && t->seqs <= kMaxRows && t->max_pages >= 1,
             "seqs must be in [1, %d] and max_pages >= 1 (got %d, %d)", kMaxRows, t->seqs, t->max_pages);
  CE_REQUIRE(t->pages >= 1 && t->pages <= kMaxPages, "pages must be in [1, %d] (got %d)", kMaxPages, t->pages);
  CE_REQUIRE(t->page_size >= 1 && t->page_size <= kMaxPage && (t->page_size & (t->page_size - 1)) == 0,
             "page_size must be a power of two in [1, %d] (got %d)", kMaxPage, t->page_size);
  CE_REQUIRE((int64_t)t->max_pages * t->page_size <= 0x7fffffff, "max_pages * page_size must be below 2^31");
  return CE_OK;
}

}  // namespace paged

using namespace paged;

// Reads and clears the status word of the table and append kernels.
int paged_status() {
  CE_CUDA_TRY(cudaDeviceSynchronize());
  DeviceStatus h{};
  CE_CUDA_TRY(cudaMemcpyFromSymbol(&h, g_paged_status, sizeof(h)));
  if (h.code == 0) return CE_OK;
  const DeviceStatus zero{};
  CE_CUDA_TRY(cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(zero)));
  return set_error(CE_ERR_USAGE, h.where == kSiteSlot  ? "paged append: a slot lies past the pool"
                                 : h.where == kSitePos ? "paged append: a position lies past the rotary table"
                                 : h.where == kSitePage ? "block table: a page id lies outside the pool"
                                                        : "block table: a length does not fit its row");
}

}  // namespace ce

using namespace ce;

extern "C" {

int ce_paged_resize(const ce_page_table *to, const ce_page_table *from, const int32_t *new_lens, int64_t *slots,
                    int32_t *pos, int capacity, int32_t *starts, int32_t *status, ce_stream_t stream) {
  int rc = check_pair(to, from);
  if (rc != CE_OK) return rc;
  CE_REQUIRE(new_lens != nullptr, "null new lengths");
  CE_REQUIRE(capacity >= 0 && (capacity == 0 || (slots != nullptr && pos != nullptr)),
             "slots and pos are required for a capacity of %d", capacity);
  CE_REQUIRE(capacity <= kMaxCapacity, "capacity must be at most %d (got %d)", kMaxCapacity, capacity);
  rc = configure_tables();
  if (rc != CE_OK) return rc;
  const int ranks = resize_ranks(from, capacity);
  const ResizeArgs a = {tables_of(to, from, status), new_lens, slots, pos, starts, capacity};
  return launch_tables(resize_kernel, a, ranks, table_smem(from, ranks), (cudaStream_t)stream, "resize_kernel");
}

int ce_paged_reorder(const ce_page_table *to, const ce_page_table *from, const int32_t *parents, int beams,
                     const ce_paged_kv *kv, int32_t *copies, int32_t *status, ce_stream_t stream) {
  int rc = check_pair(to, from);
  if (rc != CE_OK) return rc;
  CE_REQUIRE(to->table_dev != from->table_dev, "the tables of `to` and `from` must differ");
  CE_REQUIRE(parents != nullptr && copies != nullptr, "null parents or copies");
  CE_REQUIRE(beams >= 1 && from->seqs % beams == 0, "%d rows are no whole number of groups of %d", from->seqs, beams);
  if (kv != nullptr) {
    rc = check_kv(kv, 0);
    if (rc != CE_OK) return rc;
    CE_REQUIRE(kv->pages == from->pages && kv->page_size == from->page_size,
               "the cache has %d pages of %d, the block table %d of %d", kv->pages, kv->page_size, from->pages,
               from->page_size);
  }
  // 16-byte pieces of a page's tokens in one layer, at most
  const long long most =
      kv != nullptr ? (kv->page_size - 1ll) * kv->kv_heads * (kv->head_dim * type_bytes(kv->type) / 16) : 0;
  CE_REQUIRE(most < (1ll << 30), "a page of a layer is too large (%d tokens, %d heads)", kv->page_size, kv->kv_heads);
  rc = configure_tables();
  if (rc != CE_OK) return rc;
  const cudaStream_t s = (cudaStream_t)stream;
  const int ranks = reorder_ranks(from);
  const ReorderArgs a = {tables_of(to, from, status), parents, beams, copies};
  rc = launch_tables(reorder_kernel, a, ranks, table_smem(from, ranks), s, "reorder_kernel");
  if (rc != CE_OK || kv == nullptr || kv->page_size == 1) return rc;
  const int b = type_bytes(kv->type);
  const CopyArgs c = {copies, to->lens_dev, static_cast<char *>(kv->k_dev), static_cast<char *>(kv->v_dev),
                      kv->layer_stride * b, kv->page_stride * b, kv->head_stride * b, kv->token_stride * b,
                      from->seqs, kv->layers, kv->kv_heads, kv->head_dim * b / 16, kv->page_size};
  const long long pairs = (long long)from->seqs * kv->layers, ctas = 8ll * sm_count();
  const unsigned x = (unsigned)std::min(pairs, ctas);
  const unsigned y = (unsigned)std::max(1ll, std::min(ctas / x, most / (4 * kCopyThreads)));
  return launch_kernel(copy_pages_kernel, dim3(x, y), dim3(kCopyThreads), 0, s, true, "copy_pages_kernel", c);
}

int ce_paged_append(const ce_paged_kv *kv, int layer, void *q_out, int q_out_type, const void *q, const void *k,
                    const void *v, int in_type, int64_t q_ld, int64_t k_ld, int64_t v_ld, const int64_t *slots,
                    const int32_t *pos, int tokens, int heads, const float *rope, int rope_len, ce_stream_t stream) {
  const int rc = check_kv(kv, layer);
  if (rc != CE_OK) return rc;
  CE_REQUIRE(tokens >= 0, "tokens must be >= 0 (got %d)", tokens);
  if (tokens == 0) return CE_OK;
  CE_REQUIRE(k != nullptr && v != nullptr && slots != nullptr, "null k, v or slots");
  CE_REQUIRE((q == nullptr) == (q_out == nullptr), "q and q_out come together");
  CE_REQUIRE(in_type == CE_TYPE_F32 || type16(in_type), "q, k, v must be F32, BF16 or F16 (got %d)", in_type);
  CE_REQUIRE(q == nullptr || type16(q_out_type), "q_out must be BF16 or F16 (got %d)", q_out_type);
  CE_REQUIRE(q == nullptr || heads >= 1, "heads must be >= 1 (got %d)", heads);
  CE_REQUIRE(rope == nullptr || (pos != nullptr && rope_len >= 1), "a rotary table needs positions and rope_len >= 1");
  const int64_t unit = 16 / type_bytes(in_type), dim = kv->head_dim;
  CE_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(rope) && q_ld % unit == 0 &&
                 k_ld % unit == 0 && v_ld % unit == 0,
             "q, k, v, q_out and rope must be 16-byte aligned, their row strides multiples of 16 bytes");
  CE_REQUIRE((q == nullptr || q_ld >= heads * dim) && k_ld >= kv->kv_heads * dim && v_ld >= kv->kv_heads * dim,
             "a row stride is shorter than its heads");
  const int b = type_bytes(kv->type);
  AppendArgs a = {};
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.kc = static_cast<char *>(kv->k_dev) + (long long)layer * kv->layer_stride * b;
  a.vc = static_cast<char *>(kv->v_dev) + (long long)layer * kv->layer_stride * b;
  a.k_scale = kv->k_scale_dev, a.v_scale = kv->v_scale_dev;
  a.slots = slots, a.pos = pos, a.rope = rope;
  a.q_ld = q_ld, a.k_ld = k_ld, a.v_ld = v_ld;
  a.page_stride = kv->page_stride, a.head_stride = kv->head_stride, a.token_stride = kv->token_stride;
  a.slot_end = (long long)kv->pages * kv->page_size;
  a.tokens = tokens, a.heads = q != nullptr ? heads : 0, a.kv_heads = kv->kv_heads, a.dim = kv->head_dim;
  a.shift = log2_of(kv->page_size), a.rope_len = rope_len;
  const unsigned x = (unsigned)a.dim / 8, y = kAppendThreads / x;
  const long long all = a.heads + 2ll * a.kv_heads;
  CE_REQUIRE(all <= 65535ll * y, "too many heads (%d + 2 x %d)", heads, kv->kv_heads);
  const dim3 grid((unsigned)tokens, (unsigned)((all + y - 1) / y)), block(x, y);
  const cudaStream_t s = (cudaStream_t)stream;
  if (in_type == CE_TYPE_F32) return launch_append<float>(q_out_type, kv->type, a, grid, block, s);
  if (in_type == CE_TYPE_F16) return launch_append<__half>(q_out_type, kv->type, a, grid, block, s);
  return launch_append<__nv_bfloat16>(q_out_type, kv->type, a, grid, block, s);
}

}  // extern "C"
