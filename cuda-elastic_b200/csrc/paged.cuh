// Shared parts of the paged key-value cache operators (paged.cu,
// paged_attention.cu) and the beam search selection (beam.cu): argument
// checks, element conversion and the status word of the paged kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace ce {
namespace paged {

constexpr int kMaxRows = 8192;       // rows of a block table
constexpr int kMaxPages = 1 << 20;   // pages of a pool
constexpr int kMaxPage = 1024;       // tokens of a page

// Sites recorded by report_timeout in the status word (ce_device_status).
constexpr unsigned kSiteSlot = 950;  // slot past the pool
constexpr unsigned kSitePos = 951;   // position past the rotary table
constexpr unsigned kSitePage = 952;  // page id outside the pool
constexpr unsigned kSiteLen = 953;   // length outside the table's row
constexpr unsigned kSiteWait = 954;  // a bounded wait for a copy gave up

inline bool type16(int t) { return t == CE_TYPE_BF16 || t == CE_TYPE_F16; }
inline int type_bytes(int t) { return t == CE_TYPE_F32 ? 4 : t == CE_TYPE_E4M3 ? 1 : 2; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

int check_kv(const ce_paged_kv *kv, int layer);        // pool and layer (CE_REQUIRE style)
int check_table(const ce_page_table *t, const char *what);

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T warp_inclusive_sum(T x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Inclusive sum over the block of one value per thread; `total` is the
// block's sum. scratch: one word per warp, free for reuse after the call.
template <typename T>
__device__ __forceinline__ T block_inclusive_sum(T v, T *scratch, T &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T x = warp_inclusive_sum(v);
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  const T ends = warp_inclusive_sum(lane < warps ? scratch[lane] : T(0));
  total = __shfl_sync(0xffffffffu, ends, 31);
  const T before = __shfl_sync(0xffffffffu, ends, warp > 0 ? warp - 1 : 0);
  __syncthreads();
  return (warp > 0 ? before : T(0)) + x;
}

__device__ __forceinline__ int add_acq_rel(int *p, int v) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// First index of [0, n) whose value is above x (n if none); a ascending.
__device__ __forceinline__ int first_above(const int *a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

}  // namespace paged
}  // namespace ce
