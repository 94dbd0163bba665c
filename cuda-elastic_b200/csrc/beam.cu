// Beam search selection: the best tokens of each beam, then the best beams x
// tokens of each batch element.
#include <float.h>

#include "paged.cuh"

namespace ce {
namespace paged {
namespace {

constexpr int kMaxBeams = 32;

struct BeamArgs {
  float *scores_out;
  int32_t *parents, *tokens;
  uint8_t *finished_out;
  const void *logits;
  long long ld;
  const float *scores;
  const uint8_t *finished;
  int batch, beams, vocab, eos, pad;
  unsigned long long *best;  // [rows][beams]
  float *lse;                // [rows]
};

// A logit as the selection takes it: NaN is -inf, +inf the largest finite
// value, -0 is +0.
template <typename T>
__device__ __forceinline__ float logit_of(T v) {
  const float x = to_float(v);
  return x != x ? -INFINITY : fminf(x, FLT_MAX) + 0.f;
}

// Keys order tokens by (logit descending, token ascending) as integers.
__device__ __forceinline__ unsigned long long key_of(float x, int token) {
  const uint32_t b = __float_as_uint(x);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((unsigned long long)o << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_token(unsigned long long k) { return (int)~(uint32_t)k; }

template <typename T>
__device__ __forceinline__ T block_reduce_max(T v, T *scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const T y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y > v ? y : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v = scratch[w] > v ? scratch[w] : v;
  return v;
}

// One CTA per beam: its log sum, then its best tokens one after the other.
template <typename T>
__global__ void __launch_bounds__(256) rows_kernel(BeamArgs a) {
  __shared__ unsigned long long best8[8];
  __shared__ float red[8];
  const int row = blockIdx.x;
  const T *x = static_cast<const T *>(a.logits) + row * a.ld;
  pdl_launch_dependents();
  pdl_wait();
  if (a.finished[row]) return;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) m = fmaxf(m, logit_of(x[i]));
  m = block_reduce_max(m, red);
  float sum = 0.f;
  if (m > -INFINITY)
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) sum += expf(logit_of(x[i]) - m);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) sum += red[w];
    a.lse[row] = m + logf(sum);
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < min(a.beams, a.vocab); ++r) {
    unsigned long long k = 0;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
      const unsigned long long c = key_of(logit_of(x[i]), i);
      if (c < last && c > k) k = c;
    }
    last = block_reduce_max(k, best8);
    if (threadIdx.x == 0) a.best[(size_t)row * a.beams + r] = last;
  }
}

// One warp per batch element: lane k walks down beam k's sorted offers.
__global__ void __launch_bounds__(32) groups_kernel(BeamArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x, lane = threadIdx.x, row = g * a.beams + lane;
  const bool beam = lane < a.beams;
  const bool done = beam && a.finished[row] != 0;
  float base = beam ? a.scores[row] : 0.f;
  const float lse = beam && !done ? a.lse[row] : 0.f;
  const int offers = !beam ? 0 : done ? 1 : min(a.beams, a.vocab);
  int at = 0, token = a.pad;
  float score = base;
  auto load = [&] {
    if (!done && at < offers) {
      const unsigned long long k = a.best[(size_t)row * a.beams + at];
      const float x = key_logit(k);
      token = key_token(k);
      score = x == -INFINITY ? -INFINITY : base + (x - lse);
    }
    if (score != score) score = -INFINITY;
  };
  load();
  for (int r = 0; r < a.beams; ++r) {
    // the best head; ties go to the lowest beam
    unsigned long long k = at < offers ? key_of(score + 0.f, lane) : 0ull;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long y = __shfl_xor_sync(0xffffffffu, k, o);
      k = y > k ? y : k;
    }
    if (lane == key_token(k)) {
      const size_t to = (size_t)g * a.beams + r;
      a.scores_out[to] = score;
      a.parents[to] = lane;
      a.tokens[to] = token;
      a.finished_out[to] = done || token == a.eos;
      ++at;
      load();
    }
  }
}

}  // namespace
}  // namespace paged
}  // namespace ce

using namespace ce;
using namespace ce::paged;

extern "C" {

int ce_beam_workspace(int batch, int beams, int vocab, size_t *bytes) {
  CE_REQUIRE(batch >= 1 && beams >= 1 && beams <= kMaxBeams && vocab >= 1,
             "batch and vocab must be >= 1 and beams in [1, %d] (got %d, %d, %d)", kMaxBeams, batch, vocab, beams);
  CE_REQUIRE(bytes != nullptr, "null argument");
  *bytes = (size_t)batch * beams * (8 * beams + 8);
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
  CE_REQUIRE(ld >= vocab, "the row stride %lld is shorter than the vocabulary %d", (long long)ld, vocab);
  CE_REQUIRE((int64_t)batch * beams <= 0x7fffffff / 32, "batch x beams is too large (%d x %d)", batch, beams);
  CE_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
             "the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  const size_t rows = (size_t)batch * beams;
  BeamArgs a = {scores_out, parents, tokens, finished_out, logits, ld, scores, finished, batch, beams, vocab, eos, pad,
                static_cast<unsigned long long *>(workspace), nullptr};
  a.lse = reinterpret_cast<float *>(a.best + rows * beams);
  const cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto kernel) {
    return launch_kernel(kernel, dim3((unsigned)rows), dim3(256), 0, s, true, "rows_kernel", a);
  };
  const int r = type == CE_TYPE_F32 ? go(rows_kernel<float>) : type == CE_TYPE_F16 ? go(rows_kernel<__half>)
                                                                                   : go(rows_kernel<__nv_bfloat16>);
  if (r != CE_OK) return r;
  return launch_kernel(groups_kernel, dim3((unsigned)batch), dim3(32), 0, s, true, "groups_kernel", a);
}

}  // extern "C"
