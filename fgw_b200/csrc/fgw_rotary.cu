// Rotary positions and cache append of a ragged batch of new tokens (fgw_rotary_append in include/fgw_mha.h).
//
// Token t, the i-th of request b's n new ones, has position p = len[b] - n + i. Each pair (x, y) of the first `rotary`
// values of a head turns by the table's angle, (x cos - y sin, y cos + x sin), in FP32 and rounded once; the pair is
// values (i, i + rotary / 2) or, interleaved, (2 i, 2 i + 1); the other values pass. Queries go to `out`, keys and
// values to the cache row of position p, so the rotated keys are written once, where attention reads them.
//
// Bound by HBM: every value is read and written once (16-byte accesses; the angles of a token, `rotary` floats, are
// read once per CTA and kept in registers across the heads). A CTA finds a token's request with a 32-ary search over
// the offsets, so a large batch costs two or three loads in a row, not log2(batch). What kept it from the memory's rate
// was loads in flight: the first form, two heads at a time after the places were known, took 51.0 us for 219 MB; three
// heads, loaded while the places are found or the batch before is turned, 43.4 us; CTAs of 128 threads instead of 256,
// so that more of them are at different points, 40.8 us (5.4 TB/s). Rotary parts whose halves are no whole 16-byte chunks
// go value by value, which the instructions bound: 8192 tokens, 32 heads on 8 of 96, 24 rotated in halves 188 us, where
// adjacent pairs, which keep the chunks, take 31.6.
#include <algorithm>

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace fgw {

constexpr int kRotaryThreads = 128;
constexpr int kRotaryTokens = 4;  // at most, per CTA
constexpr int kRotaryHeads = 3;   // heads a thread loads together, one such batch ahead of the one it turns

struct RotaryArgs {
  const void *q, *k, *v;
  void *out, *k_cache, *v_cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const float* cos_sin;
  long long q_stride, k_stride, v_stride, out_stride;  // elements from token to token
  long long tokens, pool_pages;
  int batch, width, page, heads, kv_heads, dim, rotary, positions, per_cta;
  int vector_angles;  // rows of cos_sin and their halves start on 16 bytes
};

struct TokenPlace {
  int position;     // -1: none (rows outside every request or outside the tables): zeros, nothing appended
  long long row;    // cache row, -1: none
};

__device__ __forceinline__ TokenPlace token_place(const RotaryArgs& a, long long t, int lane) {
  TokenPlace p = {-1, -1};
  const int b = find_request(a.cu, a.batch, t, lane);
  const long long first = a.cu[b], last = a.cu[b + 1];
  const long long position = a.lens[b] - last + t;
  if (t < first || t >= last || position < 0 || position >= a.positions ||
      position >= static_cast<long long>(a.width) * a.page) {
    return p;
  }
  p.position = static_cast<int>(position);
  const int in_page = p.position % a.page;
  const long long id = a.table[static_cast<long long>(b) * a.width + p.position / a.page];
  if (id >= 0 && id < a.pool_pages) p.row = id * a.page + in_page;
  return p;
}

// Head h of the token: queries, then keys, then values.
template <typename T>
__device__ __forceinline__ const T* head_source(const RotaryArgs& a, long long t, int h) {
  if (h < a.heads) return static_cast<const T*>(a.q) + t * a.q_stride + static_cast<long long>(h) * a.dim;
  h -= a.heads;
  if (h < a.kv_heads) return static_cast<const T*>(a.k) + t * a.k_stride + static_cast<long long>(h) * a.dim;
  return static_cast<const T*>(a.v) + t * a.v_stride + static_cast<long long>(h - a.kv_heads) * a.dim;
}
// Where it goes (nullptr: nowhere).
template <typename T>
__device__ __forceinline__ T* head_target(const RotaryArgs& a, const TokenPlace& p, long long t, int h) {
  if (h < a.heads) return static_cast<T*>(a.out) + t * a.out_stride + static_cast<long long>(h) * a.dim;
  if (p.row < 0) return nullptr;
  h -= a.heads;
  const bool key = h < a.kv_heads;
  return static_cast<T*>(key ? a.k_cache : a.v_cache) + (p.row * a.kv_heads + (key ? h : h - a.kv_heads)) * a.dim;
}

template <typename T>
__device__ __forceinline__ void turn_pair(float& x, float& y, float c, float s) {
  const float u = x * c - y * s;
  y = y * c + x * s;
  x = u;
}

// kLayout 0: adjacent pairs; 1: pairs half the rotary part apart, in whole 16-byte chunks; 2: the same for other
// halves, value by value.
template <typename T, int kLayout>
__global__ void __launch_bounds__(kRotaryThreads) rotary_append_kernel(const RotaryArgs a) {
  using Tr = ElemTraits<T>;
  __shared__ TokenPlace places[kRotaryTokens];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long first = static_cast<long long>(blockIdx.x) * a.per_cta;
  const int count = static_cast<int>(min(static_cast<long long>(a.per_cta), a.tokens - first));
  auto find_places = [&]() {
    if (warp < count) {
      const TokenPlace p = token_place(a, first + warp, lane);
      if (lane == 0) places[warp] = p;
    }
    __syncthreads();
  };
  const int half = a.rotary / 2;
  const int all_heads = a.heads + 2 * a.kv_heads;
  if constexpr (kLayout == 2) {
    find_places();
    const int per_head = half + a.dim - a.rotary;  // pairs, then the values that pass
    for (int k = 0; k < count; ++k) {
      const TokenPlace p = places[k];
      const float* angles = a.cos_sin + static_cast<long long>(max(p.position, 0)) * a.rotary;
      for (int i = threadIdx.x; i < all_heads * per_head; i += kRotaryThreads) {
        const int e = i % per_head;
        const int h = i / per_head;
        const T* src = head_source<T>(a, first + k, h);
        T* dst = head_target<T>(a, p, first + k, h);
        if (dst == nullptr) continue;
        if (e >= half) {
          dst[half + e] = p.position < 0 ? Tr::from_float(0.f) : src[half + e];
          continue;
        }
        float x = static_cast<float>(src[e]), y = static_cast<float>(src[half + e]);
        if (h < a.heads + a.kv_heads) turn_pair<T>(x, y, angles[e], angles[half + e]);
        dst[e] = Tr::from_float(p.position < 0 ? 0.f : x);
        dst[half + e] = Tr::from_float(p.position < 0 ? 0.f : y);
      }
    }
    return;
  }
  // One slot of a head per thread: a chunk of eight values, or with kLayout 1 the two chunks of eight pairs.
  const int pair_slots = kLayout == 1 ? half / 8 : 0;
  const int slots = a.dim / 8 - pair_slots;
  const int groups = kRotaryThreads / slots;
  const int slot = threadIdx.x % slots, group = threadIdx.x / slots;
  const bool two = slot < pair_slots;
  const int at0 = two ? slot : slot + pair_slots;  // chunk within the head
  const int at1 = at0 + pair_slots;                // its partner (two)
  // The rows' values do not depend on their place, so a batch of heads is loaded while the places are found, or the
  // batch before is turned and stored.
  const int batches = (all_heads + groups * kRotaryHeads - 1) / (groups * kRotaryHeads);
  uint4 x[kRotaryHeads], y[kRotaryHeads];
  auto load = [&](int k, int batch) {
#pragma unroll
    for (int u = 0; u < kRotaryHeads; ++u) {
      const int h = group + (batch * kRotaryHeads + u) * groups;
      if (group >= groups || h >= all_heads) continue;
      const uint4* src = reinterpret_cast<const uint4*>(head_source<T>(a, first + k, h));
      x[u] = src[at0];
      if (two) y[u] = src[at1];
    }
  };
  load(0, 0);
  find_places();
  if (group >= groups) return;
  for (int k = 0; k < count; ++k) {
    const TokenPlace p = places[k];
    alignas(16) float c[8], s[8];
    if (p.position >= 0) {
      const float* angles = a.cos_sin + static_cast<long long>(p.position) * a.rotary;
      if (two && a.vector_angles) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(&c[i]) = *reinterpret_cast<const float4*>(&angles[slot * 8 + i]);
          *reinterpret_cast<float4*>(&s[i]) = *reinterpret_cast<const float4*>(&angles[half + slot * 8 + i]);
        }
      } else if (two) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c[i] = angles[slot * 8 + i];
          s[i] = angles[half + slot * 8 + i];
        }
      } else if (kLayout == 0 && a.vector_angles) {
        if (slot * 4 < half) {
          *reinterpret_cast<float4*>(&c[0]) = *reinterpret_cast<const float4*>(&angles[slot * 4]);
          *reinterpret_cast<float4*>(&s[0]) = *reinterpret_cast<const float4*>(&angles[half + slot * 4]);
        }
      } else if (kLayout == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = slot * 4 + i < half;
          c[i] = in ? angles[slot * 4 + i] : 1.f;
          s[i] = in ? angles[half + slot * 4 + i] : 0.f;
        }
      }
    }
    for (int batch = 0; batch < batches; ++batch) {
      uint4 xt[kRotaryHeads], yt[kRotaryHeads];
#pragma unroll
      for (int u = 0; u < kRotaryHeads; ++u) {
        xt[u] = x[u];
        yt[u] = y[u];
      }
      if (batch + 1 < batches) {
        load(k, batch + 1);
      } else if (k + 1 < count) {
        load(k + 1, 0);
      }
#pragma unroll
      for (int u = 0; u < kRotaryHeads; ++u) {
        const int h = group + (batch * kRotaryHeads + u) * groups;
        if (h >= all_heads) continue;
        uint4* dst = reinterpret_cast<uint4*>(head_target<T>(a, p, first + k, h));
        if (dst == nullptr) continue;
        const bool turn = h < a.heads + a.kv_heads;
        uint32_t* xw = reinterpret_cast<uint32_t*>(&xt[u]);
        uint32_t* yw = reinterpret_cast<uint32_t*>(&yt[u]);
        if (p.position < 0) {
          xt[u] = yt[u] = make_uint4(0, 0, 0, 0);
        } else if (turn && two) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 xs = Tr::unpack2(xw[i]), ys = Tr::unpack2(yw[i]);
            turn_pair<T>(xs.x, ys.x, c[2 * i], s[2 * i]);
            turn_pair<T>(xs.y, ys.y, c[2 * i + 1], s[2 * i + 1]);
            xw[i] = Tr::pack2(xs.x, xs.y);
            yw[i] = Tr::pack2(ys.x, ys.y);
          }
        } else if (turn && kLayout == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (slot * 4 + i >= half) continue;
            float2 xs = Tr::unpack2(xw[i]);
            turn_pair<T>(xs.x, xs.y, c[i], s[i]);
            xw[i] = Tr::pack2(xs.x, xs.y);
          }
        }
        dst[at0] = xt[u];
        if (two) dst[at1] = yt[u];
      }
    }
  }
}

int rotary_validate(const fgw_rotary_params& p) {
  for (int r : p.reserved) {
    if (r != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.tokens < 0 || p.tokens > 0x7fffffffll || p.batch <= 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads != 0 ||
      p.table_width <= 0 || p.page_size <= 0 || p.pool_rows <= 0 || p.pool_rows % p.page_size != 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  if (p.rotary_dim < 2 || p.rotary_dim > p.head_dim || p.rotary_dim % 2 != 0 || p.positions <= 0) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  if (static_cast<long long>(p.page_size) * p.table_width > 0x7fffffffll) return FGW_ERR_INVALID_ARGUMENT;
  if (p.dtype != FGW_DTYPE_FLOAT16 && p.dtype != FGW_DTYPE_BFLOAT16) return FGW_ERR_INVALID_ARGUMENT;
  if (p.interleaved != 0 && p.interleaved != 1) return FGW_ERR_INVALID_ARGUMENT;
  if (p.tokens == 0) return FGW_OK;
  const void* data[6] = {p.q, p.k, p.v, p.q_out, p.k_cache, p.v_cache};
  for (const void* d : data) {
    if (d == nullptr || reinterpret_cast<uintptr_t>(d) % 16 != 0) return FGW_ERR_INVALID_ARGUMENT;
  }
  if (p.block_table == nullptr || p.cache_seqlens == nullptr || p.cu_seqlens_q == nullptr || p.cos_sin == nullptr) {
    return FGW_ERR_INVALID_ARGUMENT;
  }
  const long long q_row = static_cast<long long>(p.heads) * p.head_dim, kv_row = static_cast<long long>(p.kv_heads) * p.head_dim;
  const long long strides[4] = {p.q_stride, p.q_out_stride, p.k_stride, p.v_stride};
  for (int i = 0; i < 4; ++i) {
    if (strides[i] % 8 != 0 || strides[i] < (i < 2 ? q_row : kv_row)) return FGW_ERR_INVALID_ARGUMENT;
  }
  return FGW_OK;
}

template <typename T>
static cudaError_t launch_rotary_t(const RotaryArgs& a, bool interleaved, unsigned grid, cudaStream_t stream) {
  if (interleaved) {
    rotary_append_kernel<T, 0><<<grid, kRotaryThreads, 0, stream>>>(a);
  } else if (a.rotary % 16 == 0) {
    rotary_append_kernel<T, 1><<<grid, kRotaryThreads, 0, stream>>>(a);
  } else {
    rotary_append_kernel<T, 2><<<grid, kRotaryThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t launch_rotary(const fgw_rotary_params& p, int sm_count, cudaStream_t stream) {
  if (p.tokens == 0) return cudaSuccess;
  RotaryArgs a;
  a.q = p.q;
  a.k = p.k;
  a.v = p.v;
  a.out = p.q_out;
  a.k_cache = p.k_cache;
  a.v_cache = p.v_cache;
  a.table = p.block_table;
  a.lens = p.cache_seqlens;
  a.cu = p.cu_seqlens_q;
  a.cos_sin = p.cos_sin;
  a.q_stride = p.q_stride;
  a.k_stride = p.k_stride;
  a.v_stride = p.v_stride;
  a.out_stride = p.q_out_stride;
  a.tokens = p.tokens;
  a.pool_pages = p.pool_rows / p.page_size;
  a.batch = p.batch;
  a.width = p.table_width;
  a.page = p.page_size;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.dim = p.head_dim;
  a.rotary = p.rotary_dim;
  a.positions = p.positions;
  a.vector_angles = p.rotary_dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.cos_sin) % 16 == 0;
  // one token per CTA until the card is full of CTAs
  a.per_cta = static_cast<int>(std::max(1ll, std::min<long long>(kRotaryTokens, p.tokens / (8ll * sm_count))));
  const unsigned grid = static_cast<unsigned>((p.tokens + a.per_cta - 1) / a.per_cta);
  return p.dtype == FGW_DTYPE_BFLOAT16 ? launch_rotary_t<__nv_bfloat16>(a, p.interleaved != 0, grid, stream)
                                       : launch_rotary_t<__half>(a, p.interleaved != 0, grid, stream);
}

}  // namespace fgw
