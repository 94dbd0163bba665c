// Attention of one new token per request over a paged key-value cache.
#include "paged.cuh"

namespace ce {
namespace paged {
namespace {

__device__ DeviceStatus g_attention_status;

struct AttnArgs {
  const void *q;
  void *out;
  float *lse;
  const char *k, *v;  // layer base
  const float *k_scale, *v_scale;
  const int32_t *table, *lens;
  long long q_ld, out_ld;
  long long page_stride, head_stride, token_stride;  // elements
  int seqs, max_pages, pages, heads, kv_heads, dim, shift;
  float scale;
};

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  if constexpr (sizeof(T) == 1) return float(x);
  else return paged::to_float(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// One warp per (request, head): an online softmax over its positions, lane l
// holding dimensions l, l + 32, ...
template <typename Io, typename Cache>
__global__ void __launch_bounds__(32) attention_kernel(AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  const int kh = h / (a.heads / a.kv_heads);
  const long long top = (long long)a.max_pages << a.shift;
  int len = a.lens[b];
  if (len < 0 || len > top) {
    report_timeout(&g_attention_status, kSiteLen);
    len = len < 0 ? 0 : (int)top;
  }
  const float ks = a.k_scale ? a.k_scale[kh] : 1.f, vs = a.v_scale ? a.v_scale[kh] : 1.f;
  float q[4], o[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < a.dim ? as_float(static_cast<const Io *>(a.q)[b * a.q_ld + h * a.dim + d]) * ks * a.scale : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < len; ++j) {
    const int page = a.table[(size_t)b * a.max_pages + (j >> a.shift)];
    if ((unsigned)page >= (unsigned)a.pages) {
      report_timeout(&g_attention_status, kSitePage);
      continue;
    }
    const long long at = page * a.page_stride + kh * a.head_stride + (j & ((1 << a.shift) - 1)) * a.token_stride;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < a.dim) s += q[i] * as_float(reinterpret_cast<const Cache *>(a.k)[at + d]);
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base), p = expf(s - base);
    m = mn, l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < a.dim) o[i] = o[i] * f + p * as_float(reinterpret_cast<const Cache *>(a.v)[at + d]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    if (d < a.dim)
      static_cast<Io *>(a.out)[b * a.out_ld + h * a.dim + d] = from_float<Io>(len ? o[i] * vs / l : 0.f);
  }
  if (lane == 0 && a.lse) a.lse[(size_t)b * a.heads + h] = len ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace paged

using namespace paged;

int paged_attention_status() {
  CE_CUDA_TRY(cudaDeviceSynchronize());
  DeviceStatus h{};
  CE_CUDA_TRY(cudaMemcpyFromSymbol(&h, g_attention_status, sizeof(h)));
  if (h.code == 0) return CE_OK;
  const DeviceStatus zero{};
  CE_CUDA_TRY(cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero)));
  return set_error(CE_ERR_USAGE, h.where == kSitePage ? "paged attention: a page id lies outside the pool"
                                                      : "paged attention: a length does not fit its table row");
}

}  // namespace ce

using namespace ce;

extern "C" {

int ce_paged_attention_workspace(size_t *bytes) {
  CE_REQUIRE(bytes != nullptr, "null argument");
  *bytes = 16;
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
  size_t need = 0;
  rc = ce_paged_attention_workspace(&need);
  if (rc != CE_OK) return rc;
  CE_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
             "the workspace must be 16-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  AttnArgs a = {};
  const int b = type_bytes(kv->type);
  a.q = q, a.out = out, a.lse = lse;
  a.k = static_cast<const char *>(kv->k_dev) + (long long)layer * kv->layer_stride * b;
  a.v = static_cast<const char *>(kv->v_dev) + (long long)layer * kv->layer_stride * b;
  a.k_scale = kv->k_scale_dev, a.v_scale = kv->v_scale_dev;
  a.table = pt->table_dev, a.lens = pt->lens_dev;
  a.q_ld = q_ld, a.out_ld = out_ld;
  a.page_stride = kv->page_stride, a.head_stride = kv->head_stride, a.token_stride = kv->token_stride;
  a.seqs = pt->seqs, a.max_pages = pt->max_pages, a.pages = kv->pages;
  a.heads = heads, a.kv_heads = kv->kv_heads, a.dim = kv->head_dim, a.shift = log2_of(kv->page_size);
  a.scale = scale;
  const dim3 grid((unsigned)heads, (unsigned)pt->seqs);
  const cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return launch_kernel(kernel, grid, dim3(32), 0, s, true, "attention_kernel", a); };
  if (kv->type == CE_TYPE_BF16) return go(attention_kernel<__nv_bfloat16, __nv_bfloat16>);
  if (kv->type == CE_TYPE_F16) return go(attention_kernel<__half, __half>);
  return io_type == CE_TYPE_F16 ? go(attention_kernel<__half, __nv_fp8_e4m3>)
                                : go(attention_kernel<__nv_bfloat16, __nv_fp8_e4m3>);
}

}  // extern "C"
