// Attention of a ragged batch of new tokens over a paged KV cache (fgw_chunk_attention in include/fgw_mha.h).
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G] over the first vis(t) cached tokens of t's request:
// vis = len - n + i + 1 for the i-th of its n new tokens when causal, len otherwise; rows with vis <= 0 are zeros.
// One warp per (token, head): the lanes share the head's values, one key at a time with a running maximum and sum.
#include <algorithm>

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace fgw {

struct ChunkArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  long long tokens, q_stride, out_stride, pool_pages;
  int batch, heads, kv_heads, dim, width, page, causal;
  float scale_log2;
};

constexpr int kChunkWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kChunkWarps * 32) chunk_simple_kernel(const ChunkArgs a) {
  const int lane = threadIdx.x % 32;
  const long long item = static_cast<long long>(blockIdx.x) * kChunkWarps + threadIdx.x / 32;
  if (item >= a.tokens * a.heads) return;
  const long long t = item / a.heads;
  const int h = static_cast<int>(item % a.heads);
  const int hk = h / (a.heads / a.kv_heads);
  const int b = find_request(a.cu, a.batch, t, lane);
  const long long first = a.cu[b], last = a.cu[b + 1];
  const int len = min(max(a.lens[b], 0), a.width * a.page);
  long long vis = 0;
  if (t >= first && t < last) vis = a.causal ? len - last + t + 1 : len;
  float q[8], o[8], m = -INFINITY, l = 0.f;
  const int e0 = lane * 8;
  const bool on = e0 < a.dim;
  const T* qrow = static_cast<const T*>(a.q) + t * a.q_stride + static_cast<long long>(h) * a.dim;
  for (int i = 0; i < 8; ++i) {
    q[i] = on ? static_cast<float>(qrow[e0 + i]) : 0.f;
    o[i] = 0.f;
  }
  for (long long j = 0; j < vis; ++j) {
    const long long id = a.table[static_cast<long long>(b) * a.width + j / a.page];
    const long long at = ((id * a.page + j % a.page) * a.kv_heads + hk) * a.dim + e0;
    const T* krow = static_cast<const T*>(a.k) + at;
    const T* vrow = static_cast<const T*>(a.v) + at;
    float s = 0.f;
    for (int i = 0; i < 8; ++i) s += on ? q[i] * static_cast<float>(krow[i]) : 0.f;
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale_log2;
    const float next = fmaxf(m, s);
    const float keep = m == next ? 1.f : fast_exp2(m - next), p = fast_exp2(s - next);
    l = l * keep + p;
    for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + (on ? p * static_cast<float>(vrow[i]) : 0.f);
    m = next;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (on) {
    T* orow = static_cast<T*>(a.out) + t * a.out_stride + static_cast<long long>(h) * a.dim + e0;
    for (int i = 0; i < 8; ++i) orow[i] = ElemTraits<T>::from_float(o[i] * inv);
  }
}

int chunk_validate(const fgw_chunk_params& p) {
  for (int r : p.reserved) {
    if (r != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.tokens < 0 || p.tokens > 0x7fffffffll || p.batch <= 0 || p.heads <= 0 || p.kv_heads <= 0 ||
      p.heads % p.kv_heads != 0 || p.table_width <= 0 || p.page_size <= 0 || p.page_size % 16 != 0 ||
      p.pool_rows <= 0 || p.pool_rows % p.page_size != 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(p.page_size) * p.table_width > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.pool_rows > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.dtype != FGW_DTYPE_FLOAT16 && p.dtype != FGW_DTYPE_BFLOAT16) return FGW_ERR_INVALID_ARGUMENT;
  if ((p.causal != 0 && p.causal != 1) || p.wait_budget_ms < 0) return FGW_ERR_INVALID_ARGUMENT;
  if (!(p.softmax_scale > 0.f) || p.softmax_scale > 1e30f) return FGW_ERR_INVALID_ARGUMENT;
  const long long row = static_cast<long long>(p.heads) * p.head_dim;
  if (p.q_stride < row || p.q_stride % 8 != 0 || p.out_stride < row || p.out_stride % 8 != 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.heads / p.kv_heads > kMaxGroup) return FGW_ERR_UNSUPPORTED;
  return FGW_OK;
}

int chunk_validate_pointers(const fgw_chunk_params& p) {
  const void* data[4] = {p.q, p.k_cache, p.v_cache, p.out};
  for (const void* d : data) {
    if (d == nullptr || reinterpret_cast<uintptr_t>(d) % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  return p.block_table == nullptr || p.cache_seqlens == nullptr || p.cu_seqlens_q == nullptr ? FGW_ERR_INVALID_ARGUMENT
                                                                                             : FGW_OK;
}

size_t chunk_workspace_bytes(const fgw_chunk_params& p) {
  (void)p;
  return sizeof(WorkspaceHeader);
}

cudaError_t launch_chunk(const fgw_chunk_params& p, void* workspace, int sm_count, int device, cudaStream_t stream) {
  (void)sm_count;
  (void)device;
  cudaError_t err = cudaMemsetAsync(workspace, 0, sizeof(WorkspaceHeader), stream);
  if (err != cudaSuccess) return err;
  ChunkArgs a;
  a.q = p.q;
  a.k = p.k_cache;
  a.v = p.v_cache;
  a.out = p.out;
  a.table = p.block_table;
  a.lens = p.cache_seqlens;
  a.cu = p.cu_seqlens_q;
  a.tokens = p.tokens;
  a.q_stride = p.q_stride;
  a.out_stride = p.out_stride;
  a.pool_pages = p.pool_rows / p.page_size;
  a.batch = p.batch;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.dim = p.head_dim;
  a.width = p.table_width;
  a.page = p.page_size;
  a.causal = p.causal;
  a.scale_log2 = p.softmax_scale * kLog2e;
  const long long items = p.tokens * p.heads;
  const unsigned grid = static_cast<unsigned>((items + kChunkWarps - 1) / kChunkWarps);
  if (p.dtype == FGW_DTYPE_BFLOAT16) {
    chunk_simple_kernel<__nv_bfloat16><<<grid, kChunkWarps * 32, 0, stream>>>(a);
  } else {
    chunk_simple_kernel<__half><<<grid, kChunkWarps * 32, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace fgw
