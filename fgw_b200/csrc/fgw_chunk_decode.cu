// Chunk attention, decode kernel: items of at most 16 (token, query head) rows of one request and key head.
//
// Bound by HBM: each item reads its K and V once and computes 2 x 16 x D products per key, so the kernel is a stream of
// K/V tiles with little arithmetic behind it. One persistent CTA per SM: a producer warp keeps a ring of K/V tiles full
// (TMA through the page table, 192 KB in flight or in use), and each consumer warp owns 16 keys of every tile, which it
// carries alone from scores to weighted values: S = Q K^T and O += P V with m16n8k16 MMAs on the 16 rows, its own running
// maximum and sum, P kept in registers (the score accumulator's layout is the A operand's). So no warp waits for
// another until the item ends, where the warps' states are merged in a fixed order through shared memory. The tensor
// units of a tile this small would sit idle in tcgen05's 128-row form: 16 rows leave seven eighths of it empty, and
// its scores would cross TMEM twice.
//
// The work is split without a plan kernel: every CTA sums the units of all requests and finds the start of its own
// range. That costs two or three trips to L2 before the first load; a plan launch ahead of it measured 6 us more.
//
// Rows of V from the last visible key on hold whatever the ring or the page holds: the warp zeroes them, since a zero
// weight times NaN would still be NaN.
#include <algorithm>

#include "fgw_chunk.cuh"

namespace fgw {

constexpr int kDecodeMinUnits = 2;  // units a program takes at least: a piece costs a merge

template <int NB>
struct DecodeShape {
  static constexpr int kBN = chunk_decode_keys(NB);
  static constexpr int kWarps = kBN / 16;              // consumer warps
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kBlockBytes = kBN * 128;        // 64 values of every key
  static constexpr int kTileBytes = NB * kBlockBytes;  // K or V tile
  static constexpr int kStages = (192 * 1024) / (2 * kTileBytes);
  static constexpr int kDim = NB * 64;
  static constexpr int kMergeO = kStages * 2 * kTileBytes;                  // [kWarps / 2][16][kDim] floats
  static constexpr int kMergeMl = kMergeO + kWarps / 2 * 16 * kDim * 4;     // [kWarps][16] maxima, then sums
  static constexpr int kBar = kMergeMl + 2 * kWarps * 16 * 4;
  static constexpr int kFlag = kBar + 2 * kStages * 8;
  static constexpr int kBytes = kFlag + 16 + 1024;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A CTA's range of units of all items, laid out by request, row and key head.
struct DecodeCursor {
  int b, row, hk, off;   // next item and the units of it before the range
  long long u, u_end;    // units left
  long long total;       // units of all items, over so many programs
  int programs;
};

// Units of request b's items for one key head.
__device__ __forceinline__ long long request_units(const ChunkArgs& a, int b) {
  const NewTokens nt = new_tokens(a.cu, a.tokens, b);
  const int rows = item_rows(a, nt.count, true);
  const int len = held_tokens(a.lens, b, a.width, a.page);
  long long units = 0;
  for (int r = 0; r < rows; ++r) units += item_units(a, nt.count, len, r * a.tokens_per_item);
  return units;
}

// Thread t takes the t-th of kThreads equal runs of requests, so one sum over the CTA gives the total and one over the
// threads before it the run that holds the range's start, which its thread then walks.
template <int kThreads>
__device__ DecodeCursor decode_cursor(const ChunkArgs& a, long long* shared, DecodeCursor* found) {
  const int run = (a.batch + kThreads - 1) / kThreads;
  const int begin = min(static_cast<int>(threadIdx.x) * run, a.batch), end = min(begin + run, a.batch);
  long long mine = 0;
  for (int b = begin; b < end; ++b) mine += request_units(a, b);
  mine *= a.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long before = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += up;
  }
  if (lane == 31) shared[warp] = before;
  if (threadIdx.x == 0) found->u = found->u_end = 0;
  __syncthreads();
  long long total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) base = total;
    total += shared[w];
  }
  before += base - mine;  // units of the runs before this one
  const int programs = static_cast<int>(max(1ll, min(static_cast<long long>(a.programs), total / kDecodeMinUnits)));
  const int p = blockIdx.x;
  if (p < programs) {
    const long long u = program_start(total, programs, p), u_end = program_start(total, programs, p + 1);
    if (u < u_end && before <= u && u < before + mine) {
      long long left = u - before;
      int b = begin;
      long long units = request_units(a, b);
      while (left >= units * a.kv_heads) {
        left -= units * a.kv_heads;
        units = request_units(a, ++b);
      }
      const NewTokens nt = new_tokens(a.cu, a.tokens, b);
      const int len = held_tokens(a.lens, b, a.width, a.page);
      int row = 0;
      long long w = item_units(a, nt.count, len, 0);
      while (left >= w * a.kv_heads) {
        left -= w * a.kv_heads;
        ++row;
        w = item_units(a, nt.count, len, row * a.tokens_per_item);
      }
      *found = {b, row, static_cast<int>(left / w), static_cast<int>(left % w), u, u_end, total, programs};
    }
  }
  __syncthreads();
  return *found;
}

__device__ __forceinline__ bool next_segment(const ChunkArgs& a, DecodeCursor& k, ChunkSegment& s) {
  if (k.u >= k.u_end) return false;
  NewTokens nt = new_tokens(a.cu, a.tokens, k.b);
  while (k.row >= item_rows(a, nt.count, true)) {  // on to the next request with rows
    ++k.b;
    k.row = 0;
    nt = new_tokens(a.cu, a.tokens, k.b);
  }
  const int t0 = k.row * a.tokens_per_item;
  const int units = item_units(a, nt.count, held_tokens(a.lens, k.b, a.width, a.page), t0);
  const int count = static_cast<int>(min(static_cast<long long>(units - k.off), k.u_end - k.u));
  make_segment(a, s, k.b, k.hk, nt, t0, units, k.off, count);
  s.end_u = k.u - k.off + units;
  k.u += count;
  k.off += count;
  if (k.off >= units) {
    k.off = 0;
    if (++k.hk == a.kv_heads) {
      k.hk = 0;
      ++k.row;
    }
  }
  return true;
}

template <typename T, int NB>
__global__ void __launch_bounds__(DecodeShape<NB>::kThreads, 1)
    chunk_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const __grid_constant__ ChunkArgs a) {
  using S = DecodeShape<NB>;
  using Tr = ElemTraits<T>;
  constexpr int NS = S::kStages, NW = S::kWarps, BN = S::kBN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* empty = full + NS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NW);
    }
    *reinterpret_cast<volatile int*>(smem + S::kFlag) = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 0) {
    a.slots.errors[blockIdx.x] = make_int2(0, 0);
    a.slots.cuts[blockIdx.x] = {0, 0, 0, -1};
  }
  grid_dependents_launch();
  __shared__ long long scan[S::kThreads / 32];
  __shared__ DecodeCursor found;
  DecodeCursor cur = decode_cursor<S::kThreads>(a, scan, &found);
  ChunkSegment sg;

  if (warp == NW) {
    // ---------------------------------------------------------------------------------- producer
    // Lane l issues the l-th box of a tile: boxes x blocks of 64 values x {K, V}, at most 32 of them.
    const int boxes = BN / a.box_rows;
    const int which = lane / (boxes * NB);         // 0: K, 1: V, more: idle
    const int box = lane % boxes, blk = (lane / boxes) % NB;
    const uint32_t box_bytes = a.box_rows * 128;
    const uint64_t policy = l2_policy_evict_first();
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
    }
    bool ok = true;
    uint32_t st = 0, phase = 0;
    while (ok && next_segment(a, cur, sg)) {
      const int32_t* table = a.table + static_cast<long long>(sg.b) * a.width;
      for (int j = 0; j < sg.n && ok; ++j) {
        const int tok = (sg.n_begin + j) * BN + box * a.box_rows;
        const bool load = which < 2 && tok < sg.limit;
        const int row = load ? table[tok / a.page] * a.page + tok % a.page : 0;
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], phase ^ 1, a.budget_ns));
        if (!ok) {
          if (lane == 0) chunk_error(a, 70);
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[st], loads * box_bytes);
        __syncwarp();
        if (load) {
          uint8_t* dst = smem + (2 * st + which) * S::kTileBytes + blk * S::kBlockBytes + box * box_bytes;
          tma_load_3d_hint(dst, which ? &vmap : &kmap, &full[st], blk * 64, sg.hk, row, policy);
        }
        if (++st == NS) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    return;
  }

  // ------------------------------------------------------------------------------------ consumers
  float* merge_o = reinterpret_cast<float*>(smem + S::kMergeO);
  float* merge_m = reinterpret_cast<float*>(smem + S::kMergeMl);
  float* merge_l = merge_m + NW * 16;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kFlag);  // a warp's wait gave up: all leave together at the item's first barrier
  const int g = lane / 4, c2 = (lane % 4) * 2;  // accumulator rows g and g + 8, columns c2 and c2 + 1
  // ldmatrix addresses within a tile: keys of this warp as B of Q K^T (K) and, transposed, of P V (V)
  const int kkey = warp * 16 + (lane / 16) * 8 + lane % 8, kchunk = (lane / 8) % 2;
  const int vkey = warp * 16 + (lane / 8) % 2 * 8 + lane % 8, vchunk = lane / 16;
  const uint32_t base = smem_u32(smem);
  uint32_t st = 0, phase = 0;
  while (next_segment(a, cur, sg)) {
    // Q of the item's rows as A operands, straight from global memory
    uint32_t q[NB * 4][4];
    int seen[2];
    long long row_q[2], row_o[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = g + 8 * u, i = r / a.group;
      const bool valid = i < sg.count;
      seen[u] = valid ? seen_keys(a, sg, i) : 0;
      const long long head = static_cast<long long>(sg.hk * a.group + r % a.group) * a.dim;
      row_q[u] = valid ? (sg.token0 + i) * a.q_stride + head : -1;
      row_o[u] = valid ? (sg.token0 + i) * a.out_stride + head : -1;
    }
#pragma unroll
    for (int ks = 0; ks < NB * 4; ++ks) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // rows g, g + 8, then the same rows eight values on
        const int at = ks * 16 + (u / 2) * 8 + c2;
        q[ks][u] = row_q[u % 2] >= 0 && at < a.dim
                       ? __ldg(reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + row_q[u % 2] + at))
                       : 0u;
      }
    }
    float o[NB * 8][4];
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int j = 0; j < sg.n; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[st], phase, a.budget_ns))) {
        if (lane == 0) {
          chunk_error(a, 71);
          *abort_flag = 1;
        }
        break;
      }
      const int key0 = (sg.n_begin + j) * BN + warp * 16;  // this warp's first key
      const uint32_t ktile = base + 2 * st * S::kTileBytes, vtile = ktile + S::kTileBytes;
      if (key0 < sg.limit) {
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int ks = 0; ks < NB * 4; ++ks) {
          const int chunk = (ks % 4) * 2 + kchunk;
          uint32_t b[4];
          ldmatrix_x4(b, ktile + (ks / 4) * S::kBlockBytes + kkey * 128 + ((chunk ^ (kkey % 8)) * 16));
          mma_16816<T>(s[0], q[ks], b[0], b[1]);
          mma_16816<T>(s[1], q[ks], b[2], b[3]);
        }
        if (key0 + 16 > sg.limit) {
          // V rows past the last visible key
          if (lane < 16 && key0 + lane >= sg.limit) {
            uint8_t* row = smem + (2 * st + 1) * S::kTileBytes + (warp * 16 + lane) * 128;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(row + blk * S::kBlockBytes + c * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();  // the ring's next TMA write to these rows comes after
          __syncwarp();
        }
        uint32_t p[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // rows g and g + 8
          float x[4] = {s[0][2 * u], s[0][2 * u + 1], s[1][2 * u], s[1][2 * u + 1]};
          if (key0 + 16 > seen[u]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (key0 + (i / 2) * 8 + c2 + i % 2 >= seen[u]) x[i] = -INFINITY;
            }
          }
          float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float next = fmaxf(m[u], top * a.scale_log2);
          const float ref = next == -INFINITY ? 0.f : next;
          if (__any_sync(0xffffffffu, next > m[u])) {
            const float keep = fast_exp2(m[u] - ref);
            l[u] *= keep;
#pragma unroll
            for (int i = 0; i < NB * 8; ++i) {
              o[i][2 * u] *= keep;
              o[i][2 * u + 1] *= keep;
            }
          }
          m[u] = next;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = fast_exp2(fmaf(x[i], a.scale_log2, -ref));
          p[u] = Tr::pack2(x[0], x[1]);
          p[2 + u] = Tr::pack2(x[2], x[3]);
          // the sum is over the rounded weights that multiply V
          const float2 lo = Tr::unpack2(p[u]), hi = Tr::unpack2(p[2 + u]);
          l[u] += (lo.x + lo.y) + (hi.x + hi.y);
        }
#pragma unroll
        for (int d = 0; d < NB * 4; ++d) {
          const int chunk = (d % 4) * 2 + vchunk;
          uint32_t b[4];
          ldmatrix_x4_trans(b, vtile + (d / 4) * S::kBlockBytes + vkey * 128 + ((chunk ^ (vkey % 8)) * 16));
          mma_16816<T>(o[2 * d], p, b[0], b[1]);
          mma_16816<T>(o[2 * d + 1], p, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == NS) {
        st = 0;
        phase ^= 1;
      }
    }
    // ---- the warps' states as one: common maximum, scaled sums, then O pairwise in a fixed order
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      if (lane % 4 == 0) {
        merge_m[warp * 16 + g + 8 * u] = m[u];
        merge_l[warp * 16 + g + 8 * u] = l[u];
      }
    }
    named_barrier_sync(1, NW * 32);
    if (*abort_flag != 0) return;
    float total[2], top[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      top[u] = -INFINITY;
      for (int w = 0; w < NW; ++w) top[u] = fmaxf(top[u], merge_m[w * 16 + g + 8 * u]);
      const float ref = top[u] == -INFINITY ? 0.f : top[u];
      total[u] = 0.f;
      for (int w = 0; w < NW; ++w) {
        total[u] += merge_l[w * 16 + g + 8 * u] * fast_exp2(merge_m[w * 16 + g + 8 * u] - ref);
      }
      const float keep = fast_exp2(m[u] - ref);
#pragma unroll
      for (int i = 0; i < NB * 8; ++i) {
        o[i][2 * u] *= keep;
        o[i][2 * u + 1] *= keep;
      }
    }
#pragma unroll
    for (int half = NW / 2; half > 0; half /= 2) {
      float* mine = merge_o + (warp % half) * 16 * S::kDim;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) {
          *reinterpret_cast<float2*>(mine + g * S::kDim + i * 8 + c2) = make_float2(o[i][0], o[i][1]);
          *reinterpret_cast<float2*>(mine + (g + 8) * S::kDim + i * 8 + c2) = make_float2(o[i][2], o[i][3]);
        }
      }
      named_barrier_sync(1, NW * 32);
      if (warp < half) {
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) {
          const float2 x = *reinterpret_cast<float2*>(mine + g * S::kDim + i * 8 + c2);
          const float2 y = *reinterpret_cast<float2*>(mine + (g + 8) * S::kDim + i * 8 + c2);
          o[i][0] += x.x;
          o[i][1] += x.y;
          o[i][2] += y.x;
          o[i][3] += y.y;
        }
      }
      named_barrier_sync(1, NW * 32);
    }
    if (sg.slot < 0) {
      if (warp == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (row_o[u] < 0) continue;
          const float inv = total[u] > 0.f ? 1.f / total[u] : 0.f;
          T* out = static_cast<T*>(a.out) + row_o[u];
#pragma unroll
          for (int i = 0; i < NB * 8; ++i) {
            if (i * 8 < a.dim) {
              *reinterpret_cast<uint32_t*>(out + i * 8 + c2) = Tr::pack2(o[i][2 * u] * inv, o[i][2 * u + 1] * inv);
            }
          }
        }
      }
      continue;
    }
    // A piece: normalised O and base-2 LSE to its slot
    if (warp == 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long long at = static_cast<long long>(sg.slot) * kDecodeRows + g + 8 * u;
        const float inv = total[u] > 0.f ? 1.f / total[u] : 0.f;
        float* out = a.slots.o + at * a.dim;
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) {
          if (i * 8 < a.dim) *reinterpret_cast<float2*>(out + i * 8 + c2) = make_float2(o[i][2 * u] * inv, o[i][2 * u + 1] * inv);
        }
        if (lane % 4 == 0) a.slots.lse[at] = total[u] > 0.f ? top[u] + fast_log2(total[u]) : kEmptyLse;
      }
    }
    if (sg.starts && threadIdx.x == 0) {
      a.slots.cuts[blockIdx.x] = {sg.token0, sg.count, sg.hk, program_of(cur.total, cur.programs, sg.end_u - 1)};
    }
  }
  grid_dependency_wait();  // so that what follows this kernel follows the plan ahead of it too
}

template <typename T, int NB>
static cudaError_t launch_decode_t(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream) {
  using S = DecodeShape<NB>;
  auto kernel = chunk_decode_kernel<T, NB>;
  cudaError_t err = prepare_kernel(reinterpret_cast<const void*>(kernel), S::kBytes, device, nullptr);
  if (err != cudaSuccess) return err;
  a.box_rows = chunk_box_rows(p.page_size, S::kBN);
  CUtensorMap kmap, vmap;
  if (chunk_kv_map(&kmap, p, p.k_cache, a.box_rows) != CUDA_SUCCESS) return cudaErrorInvalidValue;
  if (chunk_kv_map(&vmap, p, p.v_cache, a.box_rows) != CUDA_SUCCESS) return cudaErrorInvalidValue;
  if (a.split) {  // the plan of the tensor kernel runs ahead; this kernel does not wait for it
    return launch_after_plan(kernel, static_cast<unsigned>(a.programs), S::kThreads, S::kBytes, stream, kmap, vmap, a);
  }
  kernel<<<a.programs, S::kThreads, S::kBytes, stream>>>(kmap, vmap, a);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_decode_nb(const fgw_chunk_params& p, const ChunkArgs& a, int device, cudaStream_t stream) {
  switch ((p.head_dim + 63) / 64) {
    case 1:
      return launch_decode_t<T, 1>(p, a, device, stream);
    case 2:
      return launch_decode_t<T, 2>(p, a, device, stream);
    case 3:
      return launch_decode_t<T, 3>(p, a, device, stream);
    default:
      return launch_decode_t<T, 4>(p, a, device, stream);
  }
}

cudaError_t launch_chunk_decode(const fgw_chunk_params& p, ChunkArgs a, int device, cudaStream_t stream) {
  return p.dtype == FGW_DTYPE_BFLOAT16 ? launch_decode_nb<__nv_bfloat16>(p, a, device, stream)
                                       : launch_decode_nb<__half>(p, a, device, stream);
}

}  // namespace fgw
