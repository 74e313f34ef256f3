// Rotary positions and cache append of a ragged batch of new tokens (fgw_rotary_append in include/fgw_mha.h).
//
// Token t, the i-th of request b's n new ones, has position p = len[b] - n + i. Each pair (x, y) of the first `rotary`
// values of a head turns by the table's angle, (x cos - y sin, y cos + x sin), in FP32 and rounded once; the pair is
// values (i, i + rotary / 2) or, interleaved, (2 i, 2 i + 1); the other values pass. Queries go to `out`, keys and
// values to the cache row of position p, so the rotated keys are written once, where attention reads them.
//
// Bound by HBM: every value is read and written once (16-byte accesses; the angles of a token, `rotary` floats, are
// read once per CTA and kept in registers across the heads). A CTA finds a token's request with a 32-ary search over
// the offsets, so a large batch costs two or three loads in a row, not log2(batch).
#include <algorithm>

#include "fgw_common.cuh"
#include "fgw_kernels.h"
#include "fgw_ragged.cuh"

namespace fgw {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 4;  // at most, per CTA
constexpr int kRotaryHeads = 2;   // heads a thread loads before it stores any

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
struct HeadRow {
  const T* src;
  T* dst;     // nullptr: nothing to write
  bool turn;  // queries and keys turn, values pass
};

template <typename T>
__device__ __forceinline__ HeadRow<T> head_row(const RotaryArgs& a, const TokenPlace& p, long long t, int h) {
  HeadRow<T> r;
  if (h < a.heads) {
    r.src = static_cast<const T*>(a.q) + t * a.q_stride + static_cast<long long>(h) * a.dim;
    r.dst = static_cast<T*>(a.out) + t * a.out_stride + static_cast<long long>(h) * a.dim;
    r.turn = true;
    return r;
  }
  h -= a.heads;
  const bool key = h < a.kv_heads;
  if (!key) h -= a.kv_heads;
  r.src = static_cast<const T*>(key ? a.k : a.v) + t * (key ? a.k_stride : a.v_stride) + static_cast<long long>(h) * a.dim;
  r.dst = p.row < 0 ? nullptr
                    : static_cast<T*>(key ? a.k_cache : a.v_cache) + (p.row * a.kv_heads + h) * a.dim;
  r.turn = key;
  return r;
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
  if (warp < count) {
    const TokenPlace p = token_place(a, first + warp, lane);
    if (lane == 0) places[warp] = p;
  }
  __syncthreads();
  const int half = a.rotary / 2;
  const int all_heads = a.heads + 2 * a.kv_heads;
  if constexpr (kLayout == 2) {
    const int per_head = half + a.dim - a.rotary;  // pairs, then the values that pass
    for (int k = 0; k < count; ++k) {
      const TokenPlace p = places[k];
      const float* angles = a.cos_sin + static_cast<long long>(max(p.position, 0)) * a.rotary;
      for (int i = threadIdx.x; i < all_heads * per_head; i += kRotaryThreads) {
        const int e = i % per_head;
        const HeadRow<T> r = head_row<T>(a, p, first + k, i / per_head);
        if (r.dst == nullptr) continue;
        if (e >= half) {
          r.dst[half + e] = p.position < 0 ? Tr::from_float(0.f) : r.src[half + e];
          continue;
        }
        float x = static_cast<float>(r.src[e]), y = static_cast<float>(r.src[half + e]);
        if (r.turn) turn_pair<T>(x, y, angles[e], angles[half + e]);
        r.dst[e] = Tr::from_float(p.position < 0 ? 0.f : x);
        r.dst[half + e] = Tr::from_float(p.position < 0 ? 0.f : y);
      }
    }
    return;
  }
  // One slot of a head per thread: a chunk of eight values, or with kLayout 1 the two chunks of eight pairs.
  const int pair_slots = kLayout == 1 ? half / 8 : 0;
  const int slots = a.dim / 8 - pair_slots;
  const int groups = kRotaryThreads / slots;
  const int slot = threadIdx.x % slots, group = threadIdx.x / slots;
  if (group >= groups) return;
  const bool two = slot < pair_slots;
  const int at0 = two ? slot : slot + pair_slots;  // chunk within the head
  const int at1 = at0 + pair_slots;                // its partner (two)
  for (int k = 0; k < count; ++k) {
    const TokenPlace p = places[k];
    float c[8], s[8];
    if (p.position >= 0) {
      const float* angles = a.cos_sin + static_cast<long long>(p.position) * a.rotary;
      if (two) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c[i] = angles[slot * 8 + i];
          s[i] = angles[half + slot * 8 + i];
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
    for (int h0 = group; h0 < all_heads; h0 += groups * kRotaryHeads) {
      uint4 x[kRotaryHeads], y[kRotaryHeads];
      HeadRow<T> rows[kRotaryHeads];
#pragma unroll
      for (int u = 0; u < kRotaryHeads; ++u) {
        const int h = h0 + u * groups;
        rows[u].dst = nullptr;
        if (h >= all_heads) continue;
        rows[u] = head_row<T>(a, p, first + k, h);
        if (rows[u].dst == nullptr) continue;
        x[u] = reinterpret_cast<const uint4*>(rows[u].src)[at0];
        if (two) y[u] = reinterpret_cast<const uint4*>(rows[u].src)[at1];
      }
#pragma unroll
      for (int u = 0; u < kRotaryHeads; ++u) {
        if (rows[u].dst == nullptr) continue;
        uint32_t* xw = reinterpret_cast<uint32_t*>(&x[u]);
        uint32_t* yw = reinterpret_cast<uint32_t*>(&y[u]);
        if (p.position < 0) {
          x[u] = y[u] = make_uint4(0, 0, 0, 0);
        } else if (rows[u].turn && two) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 xs = Tr::unpack2(xw[i]), ys = Tr::unpack2(yw[i]);
            turn_pair<T>(xs.x, ys.x, c[2 * i], s[2 * i]);
            turn_pair<T>(xs.y, ys.y, c[2 * i + 1], s[2 * i + 1]);
            xw[i] = Tr::pack2(xs.x, xs.y);
            yw[i] = Tr::pack2(ys.x, ys.y);
          }
        } else if (rows[u].turn && kLayout == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (slot * 4 + i >= half) continue;
            float2 xs = Tr::unpack2(xw[i]);
            turn_pair<T>(xs.x, xs.y, c[i], s[i]);
            xw[i] = Tr::pack2(xs.x, xs.y);
          }
        }
        reinterpret_cast<uint4*>(rows[u].dst)[at0] = x[u];
        if (two) reinterpret_cast<uint4*>(rows[u].dst)[at1] = y[u];
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
  // one token per CTA until the card is full of CTAs
  a.per_cta = static_cast<int>(std::max(1ll, std::min<long long>(kRotaryTokens, p.tokens / (8ll * sm_count))));
  const unsigned grid = static_cast<unsigned>((p.tokens + a.per_cta - 1) / a.per_cta);
  return p.dtype == FGW_DTYPE_BFLOAT16 ? launch_rotary_t<__nv_bfloat16>(a, p.interleaved != 0, grid, stream)
                                       : launch_rotary_t<__half>(a, p.interleaved != 0, grid, stream);
}

}  // namespace fgw
